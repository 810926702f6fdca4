"""GPU head norms, rotation and cache store (rxq4_qk_norm_rope) against the
definition in 64 bits (serving_reference.rope, which derives the bound)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import rxq4  # noqa: F401
from rxq4 import capi
from tests import serving_reference as ref

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def inputs(p, dtype, fused, seed=5):
    g = torch.Generator().manual_seed(seed)
    if fused:
        qkv = torch.randn((p.rows, p.heads + 2 * p.kv, p.hd), generator=g).to(dtype)
        return qkv[:, :p.heads], qkv[:, p.heads:p.heads + p.kv], qkv[:, p.heads + p.kv:], qkv
    x = [torch.randn((p.rows, n, p.hd), generator=g).to(dtype) for n in (p.heads, p.kv, p.kv)]
    return (*x, None)


def run(p, x, inv_freq, qw, kw, eps, interleaved, cache=None, batch=None, q_out=None):
    if cache is None:
        cache, batch = p.device(capi)
    q, k, v, fused = x
    if fused is not None:
        f = fused.cuda()
        q, k, v = f[:, :p.heads], f[:, p.heads:p.heads + p.kv], f[:, p.heads + p.kv:]
    else:
        q, k, v = q.cuda(), k.cuda(), v.cuda()
    t = lambda a: None if a is None else a.cuda()  # noqa: E731
    q_out = torch.full((p.rows, p.heads, p.hd), 7.0, dtype=F16, device="cuda") if q_out is None else q_out
    capi.qk_norm_rope(q_out, q, k, v, batch, cache, t(inv_freq), t(qw), t(kw), eps, interleaved)
    return q_out, cache


def near16(got, want, bound):
    got = got.astype(np.float64)
    assert (np.abs(got - want) <= bound + ref.H16 * np.abs(want) + ref.TINY16).all()


def check(p, x, got, cache, inv_freq, qw, kw, eps, interleaved):
    """q_out rows, the stored rows, and that nothing else of the cache or of q_out
    changed."""
    f = np.zeros(0, np.float32) if inv_freq is None else inv_freq.numpy()
    w = lambda a: None if a is None else a.double().numpy()  # noqa: E731
    q, k, v = (a.double().numpy() for a in x[:3])
    got = got.cpu().numpy()
    kc, vc = (t.cpu().reshape(-1, p.kv, p.hd) for t in cache.tensors[:2])
    ks, vs = (None if t is None else t.cpu().reshape(-1, p.kv).numpy() for t in cache.tensors[3:])
    k0, v0 = p.k.reshape(-1, p.kv, p.hd), p.v.reshape(-1, p.kv, p.hd)
    rest, untouched = np.ones(len(kc), bool), np.ones(p.rows, bool)
    for i, (n, m) in enumerate(zip(p.new, p.lens)):
        rows = np.arange(int(p.starts[i]), int(p.starts[i]) + n)
        untouched[rows] = False
        pos = m - n + np.arange(n)
        assert not got[rows[pos < 0]].any()
        rows, pos = rows[pos >= 0], pos[pos >= 0]
        y, bound = ref.rope(q[rows], w(qw), eps, pos, f, interleaved)
        near16(got[rows], y, bound)
        slot = p.slots(i, max(m, 0)).numpy()[pos] if len(pos) else np.zeros(0, int)
        rows, pos, slot = rows[slot >= 0], pos[slot >= 0], slot[slot >= 0]
        rest[slot] = False
        y, bound = ref.rope(k[rows], w(kw), eps, pos, f, interleaved)
        for want, b, cached, scales in ((y, bound, kc, ks), (v[rows], np.zeros_like(v[rows]), vc, vs)):
            c = cached.numpy()[slot]
            if not p.int8:
                near16(c, want, b)
                continue
            # scale: one division of a maximum off by b; a value: half a step, and
            # what the scale and the value are off
            s, top = scales[slot].astype(np.float64), np.abs(want).max(-1)
            assert (np.abs(s - top / 127) <= b.max(-1) / 127 + 2 * ref.U * top / 127 + 2.0 ** -149).all()
            off = np.abs(c * s[..., None] - want)
            assert (off <= 0.5 * s[..., None] * (1 + 2.0 ** -14) + b + 4 * ref.U * np.abs(want)).all()
            assert np.abs(c.astype(int)).max(initial=0) <= 127
    assert torch.equal(kc[rest].view(torch.int8), k0[rest].view(torch.int8))
    assert torch.equal(vc[rest].view(torch.int8), v0[rest].view(torch.int8))
    assert (got[untouched] == 7.0).all()


def freqs(n_rot, base=1e6):
    return None if n_rot == 0 else torch.tensor(base ** (-np.arange(0, n_rot, 2) / n_rot), dtype=F32)


# heads, page, int8, dtype, fused, norm, n_rot, interleaved, new, lens
CASES = [
    ((16, 2, 128), 16, False, F16, True, True, 128, False, [1], [1001]),
    ((16, 2, 128), 16, False, F16, False, True, 128, False, [1], [1]),
    ((32, 8, 128), 64, False, BF16, True, True, 128, False, [70, 1, 300], [70, 64, 1000]),
    ((32, 8, 128), 16, True, F16, True, False, 128, True, [1] * 70, [1 + 9 * i for i in range(70)]),
    ((32, 8, 128), 16, True, F32, True, True, 128, False, [33], [50]),
    ((8, 8, 64), 1, False, F32, False, True, 64, True, [5, 0, 9], [5, 9, 100]),
    ((8, 4, 80), 8, True, BF16, True, True, 32, False, [40], [64]),
    ((8, 4, 80), 8, False, F16, True, True, 40, False, [40, 1], [64, 8]),   # half a rotation of 20
    ((6, 2, 96), 32, False, F16, False, False, 24, False, [17], [40]),      # of 12
    ((6, 2, 96), 32, False, F16, False, True, 96, True, [17], [40]),
    ((4, 1, 256), 16, False, F16, True, True, 256, False, [9], [20]),
    ((4, 4, 256), 16, True, BF16, False, True, 64, True, [9], [20]),
    ((3, 1, 8), 2, False, F16, False, True, 8, False, [5], [9]),
    ((2, 2, 16), 4, True, F16, False, True, 2, False, [5], [9]),
    ((5, 1, 200), 16, False, F16, True, True, 200, False, [7], [300]),
    ((5, 1, 200), 16, False, F16, True, True, 0, False, [7], [300]),        # no rotation
    ((1, 1, 128), 16, False, BF16, True, False, 0, False, [3], [3]),        # neither
    ((64, 8, 128), 128, False, F16, True, True, 128, False, [600], [5000]),
]


@pytest.mark.parametrize("heads,page,int8,dtype,fused,norm,n_rot,interleaved,new,lens", CASES)
def test_against_64_bits(heads, page, int8, dtype, fused, norm, n_rot, interleaved, new, lens):
    print(f"qk_norm_rope {heads} page={page} int8={int8} {dtype} norm={norm} n_rot={n_rot} {interleaved} {new}", flush=True)
    p = ref.Paged(31, *heads, page, new, lens, int8)
    g = torch.Generator().manual_seed(6)
    qw, kw = ((1 + 0.2 * torch.randn(heads[2], generator=g)) for _ in range(2)) if norm else (None, None)
    x = inputs(p, dtype, fused)
    args = (freqs(n_rot), qw, kw, 1e-6, interleaved)
    got, cache = run(p, x, *args)
    check(p, x, got, cache, *args)


@pytest.mark.parametrize("which", ["q", "k"])
def test_norm_of_one_side_only(which):
    p = ref.Paged(32, 16, 4, 64, 16, [9], [30])
    w = 1 + 0.1 * torch.arange(64.0)
    args = (freqs(64), w if which == "q" else None, w if which == "k" else None, 1e-5, False)
    x = inputs(p, F16, True)
    got, cache = run(p, x, *args)
    check(p, x, got, cache, *args)


def test_padding_holes_and_positions_without_a_slot():
    """Rows of no sequence, a hole under the new tokens, more new tokens than
    positions, positions past the table."""
    p = ref.Paged(33, 8, 2, 64, 16, [20, 7, 9, 1], [60, 3, 9, 0], pad=3, lead=2, holes=[(0, 3)], apart=True)
    args = (freqs(64), None, None, 1e-6, False)
    x = inputs(p, F16, True)
    got, cache = run(p, x, *args)
    check(p, x, got, cache, *args)
    p = ref.Paged(34, 8, 2, 64, 16, [30], [64])
    p.lens, p.seq_lens = [80], p.seq_lens + 16
    got, cache = run(p, x := inputs(p, F16, False), *args)
    check(p, x, got, cache, *args)


def test_far_positions():
    """Angles of millions of turns: position 16 million, frequency 1."""
    p = ref.Paged(35, 4, 1, 64, 1024, [3], [5])
    p.lens, p.seq_lens = [2 ** 24 - 1], torch.tensor([2 ** 24 - 1], dtype=torch.int32)
    args = (freqs(64, 10000.0), None, None, 1e-6, False)
    x = inputs(p, F16, True)
    got, cache = run(p, x, *args)
    check(p, x, got, cache, *args)


def test_in_place():
    p = ref.Paged(36, 16, 2, 128, 16, [40], [100])
    x = inputs(p, F16, False)
    args = (freqs(128), torch.ones(128), torch.ones(128), 1e-6, False)
    want, _ = run(p, x, *args)
    q = x[0].cuda()
    cache, batch = p.device(capi)
    capi.qk_norm_rope(q, q, x[1].cuda(), x[2].cuda(), batch, cache, args[0].cuda(), args[1].cuda(), args[2].cuda())
    assert torch.equal(q, want)


def test_int8_rows_of_zeros_tiny_and_not_finite_values():
    p = ref.Paged(37, 2, 2, 64, 16, [6], [6], True)
    q, k, v, _ = inputs(p, F32, False)
    k[0], v[0] = 0.0, 0.0
    k[1], v[1] = 1e-44, -1e-44
    k[2, 0, 3], v[2, 1, 60] = float("inf"), float("nan")
    got, cache = run(p, (q, k, v, None), None, None, None, 0.0, False)
    slot = p.slots(0, 6)
    value = lambda c, s: (c.cpu().reshape(-1, 2, 64).float() * s.cpu().reshape(-1, 2, 1))[slot]  # noqa: E731
    kk, vv = value(cache.tensors[0], cache.tensors[3]), value(cache.tensors[1], cache.tensors[4])
    assert not kk[0].any() and not vv[0].any()
    assert (kk[1] - 1e-44).abs().max() <= 1e-44 and (vv[1] + 1e-44).abs().max() <= 1e-44
    assert torch.isnan(kk[2, 0]).all() and torch.isfinite(kk[2, 1]).all()
    assert torch.isnan(vv[2, 1]).all() and torch.isfinite(vv[2, 0]).all()
    assert torch.isfinite(kk[3:]).all() and torch.isfinite(vv[3:]).all()


def test_fp16_overflow_becomes_an_infinity():
    p = ref.Paged(38, 2, 1, 64, 16, [2], [2])
    q, k, v, _ = inputs(p, F32, False)
    q[0, 0, 0], k[1, 0, 1], v[1, 0, 2] = 1e5, -1e5, 1e5
    got, cache = run(p, (q, k, v, None), None, None, None, 0.0, False)
    slot = p.slots(0, 2)
    assert got[0, 0, 0] == float("inf")
    assert cache.tensors[0].reshape(-1, 64)[slot[1], 1] == float("-inf")
    assert cache.tensors[1].reshape(-1, 64)[slot[1], 2] == float("inf")


@pytest.mark.parametrize("starts", [[0, 5, 3], [-4, 2, 9], [0, 100000, 100001], [7, 2, 1]])
def test_starts_outside_the_rows_write_nothing_outside(starts):
    p = ref.Paged(39, 8, 2, 64, 16, [4, 5], [64, 64])
    cache, batch = p.device(capi)
    batch.tensors[0].copy_(torch.tensor(starts, dtype=torch.int32))
    x = inputs(p, F16, True)
    big = torch.full((p.rows + 20, 8, 64), 7.0, dtype=F16, device="cuda")
    run(p, x, freqs(64), None, None, 1e-6, False, cache, batch, big[10:-10])
    assert (big[:10] == 7.0).all() and (big[-10:] == 7.0).all()


def test_large_pool_offsets():
    """Slots past 4 GiB of a tensor."""
    kv, hd, page = 8, 256, 1024
    n = 2 ** 32 // (page * kv * hd * 2) + 4
    k = torch.zeros((n, page, kv, hd), dtype=F16, device="cuda")
    v = torch.zeros_like(k)
    p = ref.Paged(40, 8, kv, hd, page, [5], [1030], spare=0)
    far = p.pages
    cache = capi.PagedKV(k, v, (p.table + (n - far)).int().cuda())
    _, batch = p.device(capi)
    x = inputs(p, F16, True)
    run(p, x, freqs(256), None, None, 1e-6, False, cache, batch)
    slot = (p.slots(0, 1030)[1025:] + (n - far) * page).cuda()
    assert torch.equal(v.view(-1, kv, hd)[slot].cpu(), x[2])
    assert int((v != 0).any(-1).any(-1).sum()) == 5


@pytest.mark.parametrize("n", [65, 4096, 4100, 9000])
def test_many_sequences(n):
    """A token's sequence among more than a wave's lanes hold, some without new tokens,
    rows of no sequence around them."""
    new = [0 if i % 11 == 4 else 1 + (i % 3 == 0) for i in range(n)]
    lens = [m + i % 5 for i, m in enumerate(new)]
    p = ref.Paged(53, 1, 1, 8, 4, new, lens, lead=3, pad=5)
    args = (freqs(8), None, None, 1e-6, False)
    x = inputs(p, F16, True)
    got, cache = run(p, x, *args)
    check(p, x, got, cache, *args)


def test_captured_and_replayed_at_other_positions():
    """A captured call follows seq_lens, the table and its inputs as they are at its
    replay."""
    p = ref.Paged(54, 8, 2, 64, 16, [1, 3, 1], [200] * 3)
    cache, batch = p.device(capi)
    before = [t.clone() for t in cache.tensors[:2]]
    f = torch.zeros((p.rows, p.heads + 2 * p.kv, p.hd), dtype=F16, device="cuda")
    q, k, v = f[:, :p.heads], f[:, p.heads:p.heads + p.kv], f[:, p.heads + p.kv:]
    out = torch.full((p.rows, p.heads, p.hd), 7.0, dtype=F16, device="cuda")
    inv_freq = freqs(64).cuda()
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    capi.qk_norm_rope(out, q, k, v, batch, cache, inv_freq, stream=s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        capi.qk_norm_rope(out, q, k, v, batch, cache, inv_freq, stream=s)
    for step in range(3):
        p.lens = [1 + 50 * step, 3 + 60 * step, 17 * (step + 1)]
        batch.tensors[1].copy_(torch.tensor(p.lens, dtype=torch.int32))
        x = inputs(p, F16, True, seed=60 + step)
        f.copy_(x[3])
        for t, b in zip(cache.tensors, before):
            t.copy_(b)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            graph.replay()
        torch.cuda.synchronize()
        check(p, x, out, cache, freqs(64), None, None, 1e-6, False)


def test_two_streams_at_once():
    """Two calls into different pages of one cache, at once."""
    p = ref.Paged(55, 8, 2, 64, 16, [300, 200], [400, 200])
    args = (freqs(64), None, None, 1e-6, False)
    x = inputs(p, F16, False)
    cache, _ = p.device(capi)
    q, k, v = (t.cuda() for t in x[:3])
    out = torch.full((p.rows, p.heads, p.hd), 7.0, dtype=F16, device="cuda")
    parts = []
    for i, (a, b) in enumerate(((0, 300), (300, 500))):
        one = capi.PagedKV(*cache.tensors[:2], cache.tensors[2][i:i + 1])
        batch = capi.SeqBatch(torch.tensor([0, b - a], dtype=torch.int32, device="cuda"),
                              torch.tensor([p.lens[i]], dtype=torch.int32, device="cuda"), b - a, b - a, p.lens[i])
        parts.append((out[a:b], q[a:b], k[a:b], v[a:b], batch, one))
    inv_freq = freqs(64).cuda()
    streams = [torch.cuda.Stream() for _ in parts]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, part in zip(streams, parts):
            capi.qk_norm_rope(*part, inv_freq, stream=s)
    torch.cuda.synchronize()
    check(p, x, out, cache, *args)


@pytest.mark.parametrize("interleaved", [False, True])
def test_sines_next_to_half_turns(interleaved):
    """(1000, 0) turned by nearly pi: 1000 times a sine of 1e-4 to 2e-4, whose angle is
    its remainder's distance to half a turn.  That distance in fp32 steps next to a half
    turn is off by 2^-25 half turns, 9.4e-5 in the output; kept whole, the sine is off by
    its function's 4 units in the last place (8 u), the correction's three roundings of
    9.4e-8 and the sum's: 12 u of the value and 1e-10."""
    p = ref.Paged(56, 4, 2, 64, 16, [1], [2])  # position 1
    f = torch.tensor(np.pi * (1 + np.linspace(0.32e-4, 0.63e-4, 32)), dtype=F32)
    q, k, v, _ = inputs(p, F16, False)
    q[:] = 0.0
    at, to = (slice(0, 64, 2), slice(1, 64, 2)) if interleaved else (slice(0, 32), slice(32, 64))
    q[..., at] = 1000.0
    got, _ = run(p, (q, k, v, None), f, None, None, 0.0, interleaved)
    want = 1000.0 * np.sin(f.double().numpy())
    assert (np.abs(want) > 0.09).all()
    bound = 12 * ref.U * np.abs(want) + 1e-10 + ref.H16 * np.abs(want) + ref.TINY16
    off = np.abs(got[0, :, to].cpu().double().numpy() - want)
    assert (off <= bound).all(), (off / bound).max()


def test_output_between_its_inputs():
    """q_out right behind the values and right before the keys: no overlap."""
    p = ref.Paged(57, 8, 2, 64, 16, [9], [30])
    x = inputs(p, F16, False)
    args = (freqs(64), None, None, 1e-6, False)
    flat = torch.cat([x[2].flatten(), torch.full((9 * 8 * 64,), 7.0, dtype=F16), x[1].flatten()]).cuda()
    v, out, k = flat[:9 * 128].view(9, 2, 64), flat[9 * 128:-9 * 128].view(9, 8, 64), flat[-9 * 128:].view(9, 2, 64)
    cache, batch = p.device(capi)
    capi.qk_norm_rope(out, x[0].cuda(), k, v, batch, cache, args[0].cuda())
    check(p, x, out, cache, *args)
