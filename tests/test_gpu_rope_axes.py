"""GPU rotation on several axes (rxq4_qk_norm_rope_axes) against the definition in 64
bits (selected_reference.rope_axes, which derives the bound), and against
rxq4_qk_norm_rope where the coordinates are the cache's positions."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import rxq4  # noqa: F401
from rxq4 import capi
from tests import selected_reference as sel
from tests import serving_reference as ref
from tests.test_gpu_qk_rope import BF16, F16, F32, freqs, inputs, near16

pytestmark = pytest.mark.gpu


def run(p, x, inv_freq, positions, axis_of, qw=None, kw=None, eps=1e-6, interleaved=False, cache=None, batch=None):
    if cache is None:
        cache, batch = p.device(capi)
    q, k, v, fused = x
    if fused is not None:
        f = fused.cuda()
        q, k, v = f[:, :p.heads], f[:, p.heads:p.heads + p.kv], f[:, p.heads + p.kv:]
    else:
        q, k, v = q.cuda(), k.cuda(), v.cuda()
    t = lambda a: None if a is None else a.cuda()  # noqa: E731
    out = torch.full((p.rows, p.heads, p.hd), 7.0, dtype=F16, device="cuda")
    capi.qk_norm_rope_axes(out, q, k, v, batch, cache, t(inv_freq), t(positions), t(axis_of), t(qw), t(kw), eps, interleaved)
    return out, cache


def coords_of(p, axes, seed, lo=-50, hi=5000):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(lo, hi, (axes, p.rows), generator=g, dtype=torch.int32)


def check(p, x, got, cache, inv_freq, positions, axis_of, qw, kw, eps, interleaved):
    f = np.zeros(0, np.float32) if inv_freq is None else inv_freq.numpy()
    w = lambda a: None if a is None else a.double().numpy()  # noqa: E731
    q, k, v = (a.double().numpy() for a in x[:3])
    coords = sel.coordinates(positions.numpy(), None if axis_of is None else axis_of.numpy(), len(f))
    got = got.cpu().numpy()
    kc, vc = (t.cpu().reshape(-1, p.kv, p.hd).numpy() for t in cache.tensors[:2])
    ks = None if cache.tensors[3] is None else cache.tensors[3].cpu().reshape(-1, p.kv).numpy()
    vs = None if cache.tensors[4] is None else cache.tensors[4].cpu().reshape(-1, p.kv).numpy()
    mine, stored = np.zeros(p.rows, bool), np.zeros(len(kc), bool)
    for i, (n, m) in enumerate(zip(p.new, p.lens)):
        rows = np.arange(int(p.starts[i]), int(p.starts[i]) + n)
        mine[rows] = True
        pos = m - n + np.arange(n)
        assert not got[rows[pos < 0]].any()
        rows, pos = rows[pos >= 0], pos[pos >= 0]
        y, b = sel.rope_axes(q[rows], w(qw), eps, coords[rows], f, interleaved)
        near16(got[rows], y, b)
        slot = p.slots(i, max(m, 0)).numpy()[pos] if len(pos) else np.zeros(0, int)
        rows, slot = rows[slot >= 0], slot[slot >= 0]
        stored[slot] = True
        y, b = sel.rope_axes(k[rows], w(kw), eps, coords[rows], f, interleaved)
        for want, off, c, s in ((y, b, kc[slot], ks), (v[rows], np.zeros_like(v[rows]), vc[slot], vs)):
            if not p.int8:
                near16(c, want, off)
                continue
            s, top = s[slot].astype(np.float64), np.abs(want).max(-1)
            assert (np.abs(s - top / 127) <= off.max(-1) / 127 + 2 * ref.U * top / 127 + 2.0 ** -149).all()
            d = np.abs(c * s[..., None] - want)
            assert (d <= 0.5 * s[..., None] * (1 + 2.0 ** -14) + off + 4 * ref.U * np.abs(want)).all()
    assert (got[~mine] == 7.0).all()
    assert np.array_equal(kc[~stored].view(np.int8), p.k.reshape(-1, p.kv, p.hd).numpy()[~stored].view(np.int8))
    assert np.array_equal(vc[~stored].view(np.int8), p.v.reshape(-1, p.kv, p.hd).numpy()[~stored].view(np.int8))


# heads, page, int8, dtype, norm, n_rot, interleaved, axes, layout, new, lens
CASES = [
    ((16, 2, 128), 16, False, F16, True, 128, False, 3, "sections", [1], [1001]),
    ((32, 8, 128), 64, False, BF16, True, 128, False, 3, "turns", [70, 1, 300], [70, 64, 1000]),
    ((32, 8, 128), 16, True, F32, False, 128, True, 3, "sections", [33, 1], [50, 9]),
    ((8, 8, 64), 1, False, F32, True, 64, True, 2, "turns", [5, 0, 9], [5, 9, 100]),
    ((8, 4, 80), 8, True, BF16, True, 32, False, 4, "random", [40], [64]),
    ((6, 2, 96), 32, False, F16, False, 24, False, 16, "random", [17], [40]),
    ((4, 1, 256), 16, False, F16, True, 256, False, 3, "sections", [300], [320]),
    ((3, 1, 8), 2, False, F16, True, 8, False, 1, None, [5], [9]),
    ((2, 2, 16), 4, True, F16, True, 2, False, 2, "turns", [5], [9]),
    ((5, 1, 200), 16, False, F16, True, 0, False, 2, None, [7], [300]),  # no rotation at all
]


@pytest.mark.parametrize("heads,page,int8,dtype,norm,n_rot,interleaved,axes,layout,new,lens", CASES)
def test_against_64_bits(heads, page, int8, dtype, norm, n_rot, interleaved, axes, layout, new, lens):
    print(f"rope axes {heads} page={page} int8={int8} {dtype} n_rot={n_rot} axes={axes} {layout} {new}", flush=True)
    p = ref.Paged(51, *heads, page, new, lens, int8, pad=2, lead=1)
    g = torch.Generator().manual_seed(52)
    qw, kw = ((1 + 0.2 * torch.randn(heads[2], generator=g)) for _ in range(2)) if norm else (None, None)
    pair = torch.arange(n_rot // 2)
    axis_of = {None: None, "sections": pair * axes // max(n_rot // 2, 1), "turns": pair % axes,
               "random": torch.randint(0, axes, (n_rot // 2,), generator=g)}[layout]
    axis_of = None if axis_of is None else axis_of.int()
    x = inputs(p, dtype, True)
    args = (freqs(n_rot), coords_of(p, axes, 53), axis_of, qw, kw, 1e-6, interleaved)
    got, cache = run(p, x, *args)
    check(p, x, got, cache, *args)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("new,lens", [([1, 1], [700, 9]), ([60, 1, 9], [300, 2, 4])])
def test_the_caches_positions_give_the_other_entry_points_bits(int8, dtype, new, lens):
    """On one axis, on three alike, and with axis_of None; a sequence with fewer
    positions than new tokens among them (4 of 9)."""
    p = ref.Paged(54, 16, 4, 128, 16, new, lens, int8)
    x = inputs(p, dtype, True)
    f = freqs(128)
    pos = torch.zeros(p.rows, dtype=torch.int32)
    for i, (n, m) in enumerate(zip(new, lens)):
        pos[int(p.starts[i]):int(p.starts[i]) + n] = torch.arange(m - n, m)
    cache, batch = p.device(capi)
    want = torch.full((p.rows, 16, 128), 7.0, dtype=F16, device="cuda")
    q, k, v = (t.cuda().contiguous() for t in x[:3])
    capi.qk_norm_rope(want, q, k, v, batch, cache, f.cuda())
    three = torch.stack([pos] * 3)
    for positions, axis_of in ((pos[None], None), (three, (torch.arange(64) % 3).int()), (three, None)):
        got, other = run(p, x, f, positions, axis_of)
        assert torch.equal(got, want)
        for a, b in zip(cache.tensors, other.tensors):
            assert (a is None and b is None) or torch.equal(a.view(torch.int8), b.view(torch.int8))


def test_axes_out_of_range_and_the_ends_of_the_coordinates():
    """An axis that is none counts as coordinate 0; coordinates at the type's ends."""
    p = ref.Paged(55, 8, 2, 64, 16, [20], [60])
    axis_of = torch.tensor([0, 1, 2, 3, -1, 2 ** 31 - 1, -2 ** 31, 1] * 4, dtype=torch.int32)
    positions = coords_of(p, 3, 56)
    positions[1, ::3], positions[2, ::4] = 2 ** 31 - 1, -2 ** 31
    x = inputs(p, F16, True)
    args = (freqs(64), positions, axis_of, None, None, 1e-6, False)
    got, cache = run(p, x, *args)
    check(p, x, got, cache, *args)


def test_rows_of_positions_apart_holes_and_padding():
    p = ref.Paged(57, 8, 2, 64, 16, [20, 7, 9, 1], [60, 3, 9, 0], pad=3, lead=2, holes=[(0, 3)], apart=True)
    wide = torch.randint(0, 900, (3, p.rows + 13), dtype=torch.int32)
    axis_of = (torch.arange(32) % 3).int()
    x = inputs(p, F16, True)
    cache, batch = p.device(capi)
    q, k, v = (t.cuda().contiguous() for t in x[:3])
    out = torch.full((p.rows, 8, 64), 7.0, dtype=F16, device="cuda")
    capi.qk_norm_rope_axes(out, q, k, v, batch, cache, freqs(64).cuda(), wide.cuda()[:, :p.rows], axis_of.cuda())
    check(p, x, out, cache, freqs(64), wide[:, :p.rows], axis_of, None, None, 1e-6, False)


def test_in_place_replayed_and_on_another_stream():
    p = ref.Paged(58, 8, 2, 64, 16, [1, 30, 1], [200, 90, 64])
    cache, batch = p.device(capi)
    x = inputs(p, F16, False)
    axis_of, f = (torch.arange(32) % 3).int(), freqs(64)
    positions = coords_of(p, 3, 59)
    q, k, v = (t.cuda() for t in x[:3])
    at, axis, freq, out = positions.cuda(), axis_of.cuda(), f.cuda(), torch.empty_like(q)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        capi.qk_norm_rope_axes(out, q, k, v, batch, cache, freq, at, axis, stream=s)
    for step in range(3):
        positions = positions + 17 * step
        at.copy_(positions)
        p.lens = [m - 3 * step for m in p.lens]
        p.seq_lens = torch.tensor(p.lens, dtype=torch.int32)
        batch.tensors[1].copy_(p.seq_lens)
        fresh = ref.Paged(58, 8, 2, 64, 16, [1, 30, 1], [200, 90, 64])
        cache.tensors[0].copy_(fresh.k)
        cache.tensors[1].copy_(fresh.v)
        out.fill_(7.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            graph.replay()
        torch.cuda.synchronize()
        check(p, x, out, cache, f, positions, axis_of, None, None, 1e-6, False)
    capi.qk_norm_rope_axes(q, q, k, v, batch, cache, freq, at, axis)
    assert torch.equal(q, out)
