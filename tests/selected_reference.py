"""Rotation on several axes, bounds of pages, the choice of pages and attention over
chosen pages on the CPU, from their definitions, in 64 bits where they are not whole
numbers, with the bounds that the tests hold the GPU's results to.

Units as in serving_reference: u = 2^-24 (half a step of fp32), h = 2^-11 (of fp16)."""
from __future__ import annotations

import numpy as np
import torch

from tests.serving_reference import H16, TINY16, U, Paged


STEP = np.float32(1) / np.float32(127)  # of a largest value: the steps of a byte


def rope_axes(x, weight, eps, coords, inv_freq, interleaved):
    """serving_reference.rope with a coordinate of its own for every pair: coords
    [rows, pairs].  The same steps, so the same bound: 24 u of |a| + |b| for the angle,
    its sine and cosine, the products and their sum, hd / 8 u for the norm's sum."""
    hd = x.shape[-1]
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight
    y, size = x.copy(), np.abs(x)
    r = 2 * len(inv_freq)
    if r:
        a = np.asarray(coords, np.float64)[:, None, :] * inv_freq.astype(np.float64)
        c, s = np.cos(a), np.sin(a)
        i, j = (np.arange(0, r, 2), np.arange(1, r, 2)) if interleaved else (np.arange(r // 2), np.arange(r // 2, r))
        y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
        size[..., i] = size[..., j] = np.abs(x[..., i]) + np.abs(x[..., j])
    return y, (24 + hd / 8) * U * size


def coordinates(positions, axis_of, pairs):
    """[tokens, pairs] of positions [axes, tokens]; 0 where the axis is none."""
    axes, n = positions.shape
    axis = np.zeros(pairs, int) if axis_of is None else np.asarray(axis_of)
    inside = (axis >= 0) & (axis < axes)
    return np.where(inside[None, :], positions[np.where(inside, axis, 0)].T, 0)


def page_keys(p: Paged, page):
    """Keys of a pool page as the library widens them: fp32 [page, kv, hd]."""
    k = p.k[page].float().numpy()
    return k if p.ks is None else k * p.ks[page].numpy()[..., None]


def touched(p: Paged, max_new=None, max_len=None):
    """(page of the pool, positions held) of the pages with new tokens."""
    width = p.table.shape[1]
    limit = min(max(p.lens + [0]) if max_len is None else max_len, width * p.page)
    found = []
    for i, (n, m) in enumerate(zip(p.new, p.lens)):
        pos0 = m - n
        end = min(pos0 + (n if max_new is None else min(n, max_new)), limit)
        first = max(pos0, 0)
        for j in range(first // p.page, -(-end // p.page) if end > first else 0):
            page = int(p.table[i, j])
            if 0 <= page < p.pages:
                found.append((page, min(p.page, end - j * p.page)))
    return found


def bounds(p: Paged, page, held):
    """(int8 [kv, hd / 8, 2, 8], fp32 [kv]): the definition in fp32, where each byte
    is one IEEE division and a rounding of whole inputs."""
    k = page_keys(p, page)[:held]
    some = ~np.isnan(k).all(0)
    with np.errstate(all="ignore"):
        lo = np.where(some, np.fmin.reduce(k, 0), 0).astype(np.float32)
        hi = np.where(some, np.fmax.reduce(k, 0), 0).astype(np.float32)
        top = np.finfo(np.float32).max
        lo, hi = np.clip(lo, -top, top), np.clip(hi, -top, top)
        scale = np.maximum(np.abs(lo), np.abs(hi)).max(-1) * STEP
        step = np.where(scale > 0, scale, np.float32(1))[:, None]
        both = np.stack([np.where(scale[:, None] > 0, np.clip(np.rint(x / step), -127, 127), 0) for x in (lo, hi)], 1)
    kv, _, hd = both.shape
    return both.reshape(kv, 2, hd // 8, 8).transpose(0, 2, 1, 3).astype(np.int8), scale.astype(np.float32)


def random_bounds(seed, pages, kv, hd, spread=0.5):
    """Bounds as keys leave them, lo <= hi, the largest of a page and head 127."""
    rng = np.random.default_rng(seed)
    mid = rng.standard_normal((pages, kv, hd))
    half = 0.2 + spread * rng.random((pages, kv, hd))
    lo, hi = mid - half, mid + half
    top = np.maximum(np.abs(lo), np.abs(hi)).max(-1, keepdims=True)
    both = np.stack([np.rint(x / top * 127) for x in (lo, hi)], 2).astype(np.int8)  # pages, kv, 2, hd
    scale = (top[..., 0] / 127).astype(np.float32)
    return both.reshape(pages, kv, 2, hd // 8, 8).transpose(0, 1, 3, 2, 4).copy(), scale


def visible(p: Paged, pos, max_len=None):
    """How many pages of its sequence a token at pos sees a position of."""
    limit = min(max(p.lens + [0]) if max_len is None else max_len, p.table.shape[1] * p.page)
    sees = min(limit, pos + 1)
    return 0 if sees <= 0 else (sees - 1) // p.page + 1


def scores(q, both, scale):
    """fp32 [kv, pages]: of q [heads, hd] (fp16 values) against the bounds of a
    sequence's pages, both [pages, kv, hd / 8, 2, 8] and scale [pages, kv].  The sums
    are whole numbers; the rest are single fp32 operations."""
    pages, kv, n8 = both.shape[:3]
    q = np.nan_to_num(q.astype(np.float32), nan=0.0, posinf=65504.0, neginf=-65504.0)
    step = np.abs(q).max(-1) * STEP
    safe = np.where(step > 0, step, np.float32(1))[:, None]
    z = np.where(step[:, None] > 0, np.rint(q / safe), 0).astype(np.int64).reshape(kv, -1, n8 * 8)
    lo, hi = (both[:, :, :, i].reshape(pages, kv, n8 * 8).astype(np.float64).transpose(1, 0, 2) for i in (0, 1))
    dot = np.minimum(z, 0).astype(np.float64) @ lo.transpose(0, 2, 1) + np.maximum(z, 0).astype(np.float64) @ hi.transpose(0, 2, 1)
    with np.errstate(over="ignore"):
        s = dot.astype(np.float32) * step.reshape(kv, -1, 1) * scale.T[:, None, :]
    return s.max(1)


def select(p: Paged, both, scale, n_select, n_first, n_last, max_new=None, max_len=None):
    """int32 [rows, kv, n_select] by the definition; -7 in rows of no sequence."""
    out = np.full((p.rows, p.kv, n_select), -7, np.int32)
    for i, (n, m) in enumerate(zip(p.new, p.lens)):
        for t in range(n if max_new is None else min(n, max_new)):
            row = int(p.starts[i]) + t
            out[row] = -1
            v = visible(p, m - n + t, max_len)
            if v == 0:
                continue
            page = p.table[i, :v].numpy()
            there = (page >= 0) & (page < p.pages)
            safe = np.where(there, page, 0)
            s = scores(p.q[row].numpy(), both[safe], scale[safe])
            j = np.arange(v)
            always = (j < n_first) | (j >= v - n_last)
            for h in range(p.kv):
                rank = np.where(always, np.inf, 0)
                order = np.lexsort((j, -s[h], -rank))
                order = order[there[order]][:n_select]
                out[row, h, :len(order)] = np.sort(order)
    return out


def random_lists(p: Paged, n_select, seed, odd=True):
    """Lists for the attention: pages before the token's, its own, and (odd) -1s
    between, pages it does not see, places past the table, one page twice."""
    rng = np.random.default_rng(seed)
    out = np.full((p.rows, p.kv, n_select), -1, np.int32)
    for i, (n, m) in enumerate(zip(p.new, p.lens)):
        for t in range(n):
            v = max(visible(p, m - n + t), 0)
            for h in range(p.kv):
                row = int(p.starts[i]) + t
                k = min(n_select, v)
                pick = rng.choice(v, k, replace=False) if v else np.zeros(0, int)
                if k and rng.random() < 0.7:
                    pick[0] = v - 1
                out[row, h, :k] = np.sort(np.unique(pick)) if len(np.unique(pick)) == k else pick
                if odd:
                    out[row, h] = rng.permutation(out[row, h])
                    for bad in (-1, v, v + 3, p.table.shape[1] + 5, 2 ** 31 - 1, -2 ** 31, -2):
                        if rng.random() < 0.15:
                            out[row, h, rng.integers(n_select)] = bad
                    if n_select > 2 and rng.random() < 0.3:
                        out[row, h, 0] = out[row, h, -1]
    return out


def attend(p: Paged, lists, scale):
    """serving_reference.attend over the listed pages: outputs in 64 bits (NaN in
    rows of no sequence) and their bounds, by the same count: the positions of a page
    that is listed twice come twice into the sums."""
    out = torch.full((p.rows, p.heads, p.hd), float("nan"), dtype=torch.float64)
    bound = torch.zeros_like(out)
    group, width = p.heads // p.kv, p.table.shape[1]
    for i, (n, m) in enumerate(zip(p.new, p.lens)):
        for t in range(n):
            row, pos = int(p.starts[i]) + t, m - n + t
            v = visible(p, pos)
            for h in range(p.kv):
                entries = [int(x) for x in lists[row, h] if 0 <= x < v]
                slots = []
                for x in entries:
                    page = int(p.table[i, x]) if x < width else -1
                    if not 0 <= page < p.pages:
                        continue
                    held = min(p.page, min(pos + 1, width * p.page, max(p.lens)) - x * p.page)
                    slots += range(page * p.page, page * p.page + held)
                heads = slice(h * group, (h + 1) * group)
                if not slots:
                    out[row, heads] = 0
                    continue
                slot = torch.tensor(slots)
                at = slot // p.page, slot % p.page
                k, vv = p.k[at][:, h].double(), p.v[at][:, h].double()
                if p.ks is not None:
                    k = k * p.ks[at][:, h].double()[:, None]
                    vv = vv * p.vs[at][:, h].double()[:, None]
                q = p.q[row, heads].double()
                s = q @ k.T * scale
                size = (q.abs() @ k.abs().T * abs(scale)).amax(-1, keepdim=True).clamp(min=1)
                w = torch.softmax(s, -1)
                out[row, heads] = w @ vv
                e = (p.hd + 12) * U * size
                bound[row, heads] = 2 * (e + len(slots) * U + 2.0 ** -21) * (w @ vv.abs())
    return out, bound + H16 * out.abs() + TINY16
