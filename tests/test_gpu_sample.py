"""GPU sampling (rxq4_sample_f32) against the walk of the order in 64 bits
(serving_reference.sample): the tokens are equal.  A draw within the sums' error of
a border could go either way; sums are off by 2^-30 of the total at most here, and
no drawn number below lies that near a border."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import rxq4  # noqa: F401
from rxq4 import capi
from tests import serving_reference as ref

pytestmark = pytest.mark.gpu
F, I = torch.float32, torch.int32


def logits_of(seed, n, vocab, kind):
    r = np.random.default_rng(seed)
    if kind == "model":  # a bulk and a few raised tokens
        l = r.standard_normal((n, vocab)) * 2
        for row in l:
            row[r.integers(0, vocab, 64)] += r.random(64) * 10
    elif kind == "flat":
        l = r.standard_normal((n, vocab)) * 0.01
    elif kind == "equal":
        l = np.full((n, vocab), 1.5)
    elif kind == "few":  # many ties
        l = r.integers(-3, 4, (n, vocab)) * 0.5
    else:  # wide
        l = r.standard_normal((n, vocab)) * 300
    return l.astype(np.float32)


def run(l, u, stride=None, **params):
    n, vocab = l.shape
    dev = torch.from_numpy(l).cuda()
    if stride:
        wide = torch.full((n, stride), 1e30, dtype=F, device="cuda")
        wide[:, :vocab] = dev
        dev = wide[:, :vocab]
    ids = torch.full((n,), -7, dtype=I, device="cuda")
    t = {k: None if v is None else torch.as_tensor(np.asarray(v), dtype=I if k == "top_k" else F).cuda()
         for k, v in params.items()}
    capi.sample_f32(ids, dev, torch.as_tensor(u, dtype=F).cuda(), **t)
    return ids.cpu().numpy()


def check(l, u, stride=None, **params):
    got = run(l, u, stride, **params)
    f32 = lambda k, v: int(v) if k == "top_k" else np.float32(v)  # noqa: E731
    want = [ref.sample(l[i], np.float32(u[i]), **{k: f32(k, v[i]) for k, v in params.items() if v is not None})
            for i in range(len(l))]
    assert got.tolist() == want


@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 255, 1000, 1025, 8191, 8192, 8193, 32000, 151936, 300001])
@pytest.mark.parametrize("kind", ["model", "flat", "few"])
def test_sizes(vocab, kind):
    print(f"sample vocab={vocab} {kind}", flush=True)
    n = 4
    l = logits_of(vocab, n, vocab, kind) if vocab > 64 or kind != "model" else logits_of(vocab, n, vocab, "wide")
    u = np.random.default_rng(vocab + 1).random(n).astype(np.float32)
    check(l, u)
    check(l, u, temperature=[0.7] * n, top_k=[50] * n, top_p=[0.9] * n, min_p=[0.02] * n)


@pytest.mark.parametrize("kind", ["model", "flat", "equal", "few", "wide"])
def test_parameters(kind):
    """Every parameter alone, and mixtures of them row by row."""
    n, vocab = 24, 20011
    l = logits_of(3, n, vocab, kind)
    r = np.random.default_rng(4)
    u = r.random(n).astype(np.float32)
    pick = lambda values: r.choice(values, n)  # noqa: E731
    temperature, top_k = pick([0.0, 0.3, 0.7, 1.0, 2.5, -1.0]), pick([0, 1, 2, 40, 1000, 20011, 30000, -5])
    top_p, min_p = pick([0.0, 0.1, 0.5, 0.95, 0.9999, 1.0, 1.5]), pick([0.0, 1e-4, 0.05, 0.5, 1.0, 2.0, -1.0])
    check(l, u, temperature=temperature)
    check(l, u, top_k=top_k)
    check(l, u, top_p=top_p)
    check(l, u, min_p=min_p)
    check(l, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)


def test_the_ends_of_u():
    l = logits_of(5, 8, 5000, "few")
    u = [0.0, -1.0, 1.0, 2.0, float("nan"), np.nextafter(np.float32(1), np.float32(0)), 0.5, 1e-30]
    check(l, u, top_k=[100] * 8)
    check(l, u)


def test_equal_logits_follow_the_index():
    """All weights equal: token floor(u n), exactly."""
    n, vocab = 64, 4096
    l = np.zeros((n, vocab), np.float32)
    u = (np.arange(n) / n).astype(np.float32)
    assert run(l, u).tolist() == [vocab // n * i for i in range(n)]
    got = run(l, u, top_k=np.full(n, 64))
    assert got.tolist() == list(range(n))


def test_infinities_nan_and_the_lowest_number():
    low, inf, nan = float(np.finfo(np.float32).min), float("inf"), float("nan")
    vocab = 3000
    l = logits_of(6, 9, vocab, "model")
    l[0] = -inf                       # nothing: -1
    l[1] = nan                        # nothing: -1
    l[2] = low                        # all equal
    l[3, :2990] = -inf
    l[4, 5:2000] = low
    l[5, 17] = nan
    l[6, [40, 400, 1400]] = inf       # they share the row
    l[7], l[7, 1234] = -inf, -5.0     # one
    l[8] = -l[8] * 0 - 0.0            # zeros of both signs are equal
    l[8, ::2] = 0.0
    u = np.linspace(0.05, 0.95, 9).astype(np.float32)
    got = run(l, u)
    assert got[0] == -1 and got[1] == -1 and got[7] == 1234 and got[6] in (40, 400, 1400)
    check(l, u)
    check(l, u, temperature=[0.5] * 9, top_p=[0.9] * 9)
    check(l, u, temperature=[1e-30] * 9)
    check(l, u, temperature=[0.0] * 9)
    check(l, u, temperature=[nan] * 9)
    check(l, u, temperature=[inf] * 9, top_k=[7] * 9)


def test_rows_far_apart_and_odd():
    l = logits_of(7, 5, 1003, "model")
    check(l, [0.1, 0.3, 0.5, 0.7, 0.9], stride=1011, top_k=[10] * 5)


@pytest.mark.parametrize("rows", [1, 2, 128, 300, 1000])
def test_many_rows(rows):
    l = logits_of(8, rows, 1777, "model")
    u = np.random.default_rng(9).random(rows).astype(np.float32)
    check(l, u, temperature=[0.8] * rows, top_p=[0.95] * rows)


def test_more_rows_than_a_workspace_holds():
    """The library's large vocabulary, and rows enough for several launches."""
    n, vocab = 200, 151936
    g = torch.Generator(device="cuda").manual_seed(10)
    dev = torch.randn((n, vocab), generator=g, device="cuda") * 3
    u = torch.rand(n, generator=g, device="cuda")
    ids = torch.empty(n, dtype=I, device="cuda")
    p = torch.full((n,), 0.9, device="cuda")
    capi.sample_f32(ids, dev, u, top_p=p)
    for i in list(range(0, n, 23)) + [n - 1]:
        assert ids[i].item() == ref.sample(dev[i].cpu().numpy(), np.float32(u[i].item()), top_p=np.float32(0.9))
    one = torch.empty(1, dtype=I, device="cuda")
    for i in (0, 77, 199):  # a row does not depend on the others
        capi.sample_f32(one, dev[i:i + 1], u[i:i + 1], top_p=p[:1])
        assert one.item() == ids[i].item()


def test_repeats_and_replays():
    n, vocab = 6, 40000
    l = torch.from_numpy(logits_of(11, n, vocab, "model")).cuda()
    u = torch.rand(n, device="cuda")
    ids = torch.empty(n, dtype=I, device="cuda")
    k = torch.full((n,), 30, dtype=I, device="cuda")
    s = torch.cuda.Stream()
    capi.sample_f32(ids, l, u, top_k=k, stream=s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        capi.sample_f32(ids, l, u, top_k=k, stream=s)
    for step in range(5):
        u.uniform_()
        l.add_(torch.randn_like(l) * 0.1)
        k.fill_(5 + 10 * step)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            graph.replay()
        torch.cuda.synchronize()
        eager = torch.empty_like(ids)
        capi.sample_f32(eager, l, u, top_k=k)
        assert torch.equal(eager, ids)
        host = l.cpu().numpy()
        assert ids.tolist() == [ref.sample(host[i], np.float32(u[i].item()), top_k=5 + 10 * step) for i in range(n)]


@pytest.mark.parametrize("spread", [1e-6, 0.01, 0.05, 0.3])
def test_bins_of_thousands_of_logits(spread):
    """Borders and draws among logits that share a bin: narrowed from registers or, with
    more than they hold, from memory."""
    g = torch.Generator().manual_seed(91)
    l = (spread * torch.randn((6, 60001), generator=g)).numpy()
    u = torch.rand(6, generator=g).numpy()
    check(l, u, top_p=torch.tensor([0.2, 0.5, 0.9, 0.99, 1.0, 0.7]))
    check(l, u, top_k=torch.tensor([3000, 700, 0, 40000, 513, 5], dtype=torch.int32),
          temperature=torch.tensor([1.0, 0.5, 2.0, 1.0, 4.0, 1.0]))


def test_two_streams_at_once():
    g = torch.Generator().manual_seed(92)
    ls = [torch.randn((n, 30000), generator=g) for n in (3, 40)]
    us = [torch.rand(len(l), generator=g) for l in ls]
    on = [(torch.zeros(len(l), dtype=torch.int32, device="cuda"), l.cuda(), u.cuda()) for l, u in zip(ls, us)]
    streams = [torch.cuda.Stream() for _ in on]
    torch.cuda.synchronize()
    for _ in range(6):
        for s, args in zip(streams, on):
            capi.sample_f32(*args, stream=s)
    torch.cuda.synchronize()
    for (ids, _, _), l, u in zip(on, ls, us):
        assert ids.tolist() == [ref.sample(a, x) for a, x in zip(l.numpy(), u.numpy())]
    for s in streams:
        capi.release_workspace(s)


# What the sums may be off by, over the row's largest weight W: a weight of a slice half
# of 2^-48 of the slice's largest, a block's sum of a slice (32 of each, 512 slices at most)
# half a unit of 2^-(62 - log2 n) W, the 64-bit sums of the reference n 2^-53 of n W.
def sums_off(vocab, total):
    bits = int(vocab - 1).bit_length()
    return vocab * 2.0 ** -49 + 512 * 32 * 2.0 ** -(63 - bits) + vocab * 2.0 ** -53 * total


@pytest.mark.parametrize("vocab", [151936, 1048576, 1048577, 4194304])
def test_a_draw_among_many_small_weights(vocab):
    """One logit 16 above all others, which are equal: the token is the draw's place
    among weights of 2^-23 of the largest.  Draws are taken whose place is 0.2 tokens or
    more from the next, which is more than the sums are off."""
    top, w = 12345, np.exp(-16.0)
    total = 1 + (vocab - 1) * w
    assert 0.2 * w > sums_off(vocab, total)
    u = (np.arange(1, 4000) / 4000).astype(np.float32)
    at = (u.astype(np.float64) * total - 1) / w
    ok = np.flatnonzero((at > 1) & (at % 1 > 0.2) & (at % 1 < 0.8))
    ok = ok[::len(ok) // 20]
    u, at = u[ok], at[ok].astype(np.int64)
    l = np.zeros((1, vocab), np.float32)
    l[0, top] = 16.0
    dev = torch.from_numpy(l).cuda()
    ids = torch.empty(1, dtype=I, device="cuda")
    us = torch.from_numpy(u).cuda()
    got = []
    for i in range(len(u)):
        capi.sample_f32(ids, dev, us[i:i + 1])
        got.append(int(ids.item()))
    assert got == [int(j) + (j >= top) for j in at]


@pytest.mark.parametrize("vocab", [1048576, 1048577, 4194304])
@pytest.mark.parametrize("kind", ["model", "equal"])
def test_vocabularies_to_the_limit(vocab, kind):
    """512 slices of 2048 logits, the switch to 8192, and 512 of those."""
    print(f"sample vocab={vocab} {kind}", flush=True)
    l = logits_of(vocab, 1, vocab, kind)
    weight = float(np.exp(l[0].astype(np.float64) - l[0].max()).sum())
    off = sums_off(vocab, weight) if kind == "model" else weight * 2.0 ** -50  # (equal weights: whole numbers)
    for i, params in enumerate([dict(temperature=[0.0]), dict(top_k=[50]), dict(top_k=[100000]), dict(top_p=[0.9]),
                                dict(min_p=[0.05]), dict(temperature=[0.7], top_k=[3000], top_p=[0.95], min_p=[0.02])]):
        one = {k: int(v[0]) if k == "top_k" else np.float32(v[0]) for k, v in params.items()}
        # the first of a few draws that no error of the sums could move
        u = next(x for x in np.float32([0.13, 0.37, 0.59, 0.71, 0.83, 0.97])
                 if ref.sample_margin(l[0], x, **one) > off)
        check(l, [u], **params)


def test_repeats_and_replays_of_known_draws():
    """As above with seeded inputs, every draw and share further from a border than the
    sums are off."""
    n, vocab = 6, 40000
    g = torch.Generator().manual_seed(93)
    l = torch.from_numpy(logits_of(11, n, vocab, "model")).cuda()
    u, p = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    ids = torch.empty(n, dtype=I, device="cuda")
    k = torch.full((n,), 30, dtype=I, device="cuda")
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    capi.sample_f32(ids, l, u, top_k=k, top_p=p, stream=s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        capi.sample_f32(ids, l, u, top_k=k, top_p=p, stream=s)
    for step in range(5):
        host = l.cpu() + 0.1 * torch.randn((n, vocab), generator=g)
        l.copy_(host)
        draws, shares = torch.rand(n, generator=g), 0.5 + 0.5 * torch.rand(n, generator=g)
        u.copy_(draws)
        p.copy_(shares)
        k.fill_(5 + 2000 * step)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            graph.replay()
        torch.cuda.synchronize()
        eager = torch.empty_like(ids)
        capi.sample_f32(eager, l, u, top_k=k, top_p=p)
        assert torch.equal(eager, ids)
        rows = list(zip(host.numpy(), draws.numpy(), shares.numpy()))
        for row, x, share in rows:
            total = float(np.exp(row.astype(np.float64) - row.max()).sum())
            assert ref.sample_margin(row, x, top_k=5 + 2000 * step, top_p=share) > sums_off(vocab, total)
        assert ids.tolist() == [ref.sample(row, x, top_k=5 + 2000 * step, top_p=share) for row, x, share in rows]


@pytest.mark.parametrize("bits", [0x7F800001, 0x7FA00000, 0xFFBFFFFF, 0x7FFFFFFF, 0xFFC00001])
@pytest.mark.parametrize("vocab", [5, 1000, 9000])
def test_nan_of_every_kind(bits, vocab):
    """Signalling ones and those with a sign: as -infinity, the row's first and last logit
    and others between."""
    l = logits_of(vocab, 3, vocab, "wide") if vocab < 64 else logits_of(vocab, 3, vocab, "model")
    at = np.unique(np.array([0, vocab // 3, vocab - 1]))
    l[:, at] = np.array(bits, np.uint32).view(np.float32)
    l[2, :] = np.array(bits, np.uint32).view(np.float32)
    assert (l.view(np.uint32)[:, at] == bits).all()
    got = [run(l, [0.3, 0.9, 0.5], temperature=t) for t in (None, [0.0] * 3)]
    clean = np.where(np.isnan(l), -np.inf, l).astype(np.float32)
    for g, t in zip(got, (None, 0.0)):
        assert g.tolist() == [ref.sample(c, x, temperature=t) for c, x in zip(clean, [0.3, 0.9, 0.5])]
        assert g[2] == -1
