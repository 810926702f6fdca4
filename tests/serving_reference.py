"""The serving operators in 64 bits on the CPU, from their definitions, with the
bounds that the tests hold the GPU's results to, and inputs for them.

Units: u = 2^-24 (half a step of fp32), h = 2^-11 (half a step of fp16)."""
from __future__ import annotations

import numpy as np
import torch

U, H16 = 2.0 ** -24, 2.0 ** -11
TINY16 = 2.0 ** -25  # half a step of fp16's smallest numbers


class Paged:
    """A pool of pages in random order and a batch of sequences on it."""

    def __init__(self, seed, heads, kv, hd, page, new, lens, int8=False, scales=True, spare=2, holes=(), pad=0,
                 lead=0, apart=False):
        """holes: (sequence, page index) without a page; pad / lead: rows of no
        sequence behind / before the batch's; apart: K and V pages alternate."""
        g = torch.Generator().manual_seed(seed)
        self.heads, self.kv, self.hd, self.page, self.int8 = heads, kv, hd, page, int8
        self.new, self.lens = list(new), list(lens)
        used = [max(-(-n // page), 0) for n in lens]
        width, n = max(used + [1]), sum(used) + spare
        order = torch.randperm(n, generator=g).int()
        self.table = torch.full((len(lens), width), -1, dtype=torch.int32)
        at = 0
        for i, m in enumerate(used):
            self.table[i, :m] = order[at:at + m]
            at += m
        for i, j in holes:
            self.table[i, j] = [-1, n, 2 ** 31 - 1, -2 ** 31][(i + j) % 4]
        self.starts = torch.tensor(np.cumsum([lead] + self.new), dtype=torch.int32)
        self.rows = int(self.starts[-1]) + pad
        self.seq_lens = torch.tensor(lens, dtype=torch.int32)
        self.pages = n
        shape = (n, 2, page, kv, hd) if apart else (2, n, page, kv, hd)
        if int8:
            both = torch.randint(-127, 128, shape, generator=g).to(torch.int8)
        else:
            both = torch.randn(shape, generator=g).half()
        self.both, self.apart = both, apart
        self.ks = self.vs = None
        if int8 and scales:
            self.ks = (torch.rand((n, page, kv), generator=g) + 0.5) / 73
            self.vs = (torch.rand((n, page, kv), generator=g) + 0.5) / 73
        self.q = torch.randn((self.rows, heads, hd), generator=g).half()

    @property
    def k(self):
        return self.both[:, 0] if self.apart else self.both[0]

    @property
    def v(self):
        return self.both[:, 1] if self.apart else self.both[1]

    def slots(self, i, m):
        """Places in the pool of positions [0, m) of sequence i, -1 in holes."""
        pos = torch.arange(m)
        j = pos // self.page
        inside = j < self.table.shape[1]
        p = self.table[i].long()[j.clamp(max=self.table.shape[1] - 1)]
        ok = inside & (p >= 0) & (p < self.pages)
        return torch.where(ok, p * self.page + pos % self.page, -1)

    def device(self, capi, max_new=None, max_len=None):
        """The cache and batch descriptors on the GPU."""
        both = self.both.cuda()
        k, v = (both[:, 0], both[:, 1]) if self.apart else (both[0], both[1])
        t = lambda a: None if a is None else a.cuda()  # noqa: E731
        cache = capi.PagedKV(k, v, self.table.cuda(), t(self.ks), t(self.vs))
        batch = capi.SeqBatch(self.starts.cuda(), self.seq_lens.cuda(), self.rows,
                              max(self.new + [0]) if max_new is None else max_new,
                              max(self.lens + [0]) if max_len is None else max_len)
        return cache, batch


def attend(p: Paged, scale):
    """[rows, heads, hd] outputs in 64 bits (NaN in rows of no sequence) and the
    bound of each.

    A score is a sum of hd products in fp32, scaled: off by at most (hd + 4) u of
    the sum of its products' magnitudes.  With the maximum's subtraction and the
    exponential (8 u of 1 and the scores' own size) a weight is off by a relative
    e = (hd + 12) u S, S the row's largest such sum, at least 1; the weights' sum and
    the output's are fp32 sums of n (n u, in chunks less), the weights hold 21 bits
    or more.  Numerator and denominator together: 2 (e + n u + 2^-21) of sum p |v|.  The
    output is rounded once to fp16."""
    out = torch.full((p.rows, p.heads, p.hd), float("nan"), dtype=torch.float64)
    bound = torch.zeros_like(out)
    group = p.heads // p.kv
    for i, (n, m) in enumerate(zip(p.new, p.lens)):
        first = int(p.starts[i])
        slot = p.slots(i, max(m, 0))
        pos = torch.arange(max(m, 0))[slot >= 0]
        slot = slot[slot >= 0]
        k = p.k.reshape(-1, p.kv, p.hd)[slot].double() if not p.apart else p.k[slot // p.page, slot % p.page].double()
        v = p.v.reshape(-1, p.kv, p.hd)[slot].double() if not p.apart else p.v[slot // p.page, slot % p.page].double()
        if p.ks is not None:
            k = k * p.ks.reshape(-1, p.kv)[slot].double()[..., None]
            v = v * p.vs.reshape(-1, p.kv)[slot].double()[..., None]
        for t in range(n):
            seen = pos <= m - n + t
            if not seen.any():
                out[first + t] = 0
                continue
            q = p.q[first + t].double().view(p.kv, group, p.hd)
            kk, vv = k[seen].permute(1, 0, 2), v[seen].permute(1, 0, 2)
            s = q @ kk.transpose(1, 2) * scale
            size = (q.abs() @ kk.abs().transpose(1, 2) * abs(scale)).amax(-1, keepdim=True).clamp(min=1)
            w = torch.softmax(s, -1)
            out[first + t] = (w @ vv).view(p.heads, p.hd)
            e = (p.hd + 12) * U * size
            rel = 2 * (e + int(seen.sum()) * U + 2.0 ** -21)
            bound[first + t] = (rel * (w @ vv.abs())).view(p.heads, p.hd)
    return out, bound + H16 * out.abs() + TINY16


def rope(x, weight, eps, pos, inv_freq, interleaved):
    """x [rows, heads, hd] 64 bits: norm and rotation, and the bound before the
    output's rounding: the norm's sums and root 12 u of the value, two products and
    a sum, sine and cosine 6 u, the angle's remainder in fp32 2 u of a turn part:
    24 u of |a| + |b| covers them."""
    hd = x.shape[-1]
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight
    y, size = x.copy(), np.abs(x)
    r = 2 * len(inv_freq)
    if r:
        a = np.asarray(pos, np.float64)[:, None, None] * inv_freq.astype(np.float64)
        c, s = np.cos(a), np.sin(a)
        i, j = (np.arange(0, r, 2), np.arange(1, r, 2)) if interleaved else (np.arange(r // 2), np.arange(r // 2, r))
        y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
        both = np.abs(x[..., i]) + np.abs(x[..., j])
        size[..., i] = size[..., j] = both
    return y, (24 + hd / 8) * U * size


def sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    """One row's token in 64 bits, by walking the order."""
    l = np.where(np.isnan(logits), -np.inf, logits).astype(np.float64)
    if not (l > -np.inf).any():
        return -1
    order = np.argsort(-l, kind="stable")
    order = order[l[order] > -np.inf]
    t = 1.0 if temperature is None else float(temperature)
    if not t > 0:
        return int(order[0])
    x = l[order]
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x == x[0], 1.0, 0.0 if x[0] == np.inf else np.exp((x - x[0]) / t))
    n = len(w)
    if top_k is not None and top_k > 0:
        n = min(n, int(top_k))
    if top_p is not None and float(top_p) < 1:
        before = np.concatenate([[0.0], np.cumsum(w[:n])[:-1]])
        n = max(1, int((before < float(top_p) * w[:n].sum()).sum()))
    if min_p is not None and float(min_p) > 0:
        n = max(1, min(n, int((w >= float(min_p)).sum())))
    x = min(max(0.0 if np.isnan(u) else float(u), 0.0), 1 - 2.0 ** -24)
    c = np.cumsum(w[:n])
    return int(order[min(n - 1, int((c <= x * c[-1]).sum()))])


def sample_margin(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    """How near a row's token (of `sample`, finite logits) is to another one: the
    smallest distance of top-p's share and of the draw from a sum of weights, over the
    largest weight, and of min-p from a weight, over it."""
    if temperature is not None and not float(temperature) > 0:
        return 1.0
    x = -np.sort(-logits.astype(np.float64))
    w = np.exp((x - x[0]) / (1.0 if temperature is None else float(temperature)))
    n, near = len(w), 1.0
    if top_k is not None and top_k > 0:
        n = min(n, int(top_k))

    def border(sums, at):
        i = int(np.searchsorted(sums, at))
        return min(abs(s - at) for s in sums[max(i - 1, 0):i + 1])

    if top_p is not None and float(top_p) < 1:
        c = np.cumsum(w[:n])
        share = float(top_p) * c[-1]
        near = min(near, border(c, share))
        n = max(1, int((np.concatenate([[0.0], c[:-1]]) < share).sum()))
    if min_p is not None and float(min_p) > 0:
        near = min(near, float((abs(w[:n] - float(min_p)) / float(min_p)).min()))
        n = max(1, min(n, int((w[:n] >= float(min_p)).sum())))
    c = np.cumsum(w[:n])
    return min(near, border(c, min(max(float(u), 0.0), 1 - 2.0 ** -24) * c[-1])) if n > 1 else near
