"""How attention of a few tokens joins the chunks of a long context (rxq4_attention_paged_f16,
rxq4_attention_selected_f16), bit for bit: the rounding of each chunk's weighed part and of
the sum is part of the results that a program has had, whatever the compiler would make of it.

The parts are made exactly known: within a chunk of 128 positions all keys are alike, so that
its weights are one power of two, and the values are whole numbers whose sums are exact.
Between chunks the weights are any.  Two large chunks all but cancel, so that a rounding of
one of them shows in fp16."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import rxq4  # noqa: F401
from rxq4 import capi

pytestmark = pytest.mark.gpu
CHUNK, PAGE = 128, 16


def tree_sum(x):
    """[.., 64] by halves: lanes 32 apart first, then 16, ... 1."""
    n = 64
    while n > 1:
        n //= 2
        x = (x[..., :n] + x[..., n:2 * n]).astype(np.float32)
    return x[..., 0]


def fused(sum_, w, x):
    """One rounding, from 64 bits of mantissa: a product has 48."""
    return (sum_.astype(np.longdouble) + w.astype(np.longdouble) * x.astype(np.longdouble)).astype(np.float32)


def joined(e, parts, counts, hd):
    """The rows' outputs: e [.., chunks], parts [.., chunks, hd], counts: positions, in
    the unit of the parts.  The first two parts are fused into the sum; the others too at
    head_dim above 64, up to it product and sum are rounded each, and the last product
    once, to fp16."""
    lanes = np.zeros(e.shape[:-1] + (64,), np.float32)
    lanes[..., :e.shape[-1]] = e * counts
    inv = (np.float32(1) / tree_sum(lanes)).astype(np.float32)
    acc = np.zeros(e.shape[:-1] + (hd,), np.float32)
    for c in range(e.shape[-1]):
        w, x = e[..., c, None], parts[..., c, :]
        acc = fused(acc, w, x) if hd > 64 or c < 2 else acc + w * x
    return ((acc if hd > 64 else acc.astype(np.float64)) * inv[..., None]).astype(np.float16)


@pytest.mark.parametrize("op", ["paged", "selected"])
@pytest.mark.parametrize("hd", [48, 64, 80, 128, 200])
@pytest.mark.parametrize("chunks", [3, 4, 9, 11])
def test_chunks_are_joined_as_they_have_been(op, hd, chunks):
    rng = np.random.default_rng([hd, chunks])
    S, kv, group, n = 4, 2, 8, chunks * CHUNK
    at = rng.integers(-128, 0, (S, kv, chunks)) / 64  # a chunk's score beside each head's factor
    at[:, :, 0], at[:, :, 2] = rng.integers(-20, 0, (S, kv)) / 64, rng.integers(-100, -30, (S, kv)) / 64
    size = rng.integers(24, 64, (kv, group)) / 32
    v = rng.integers(-2, 3, (S, chunks, CHUNK, kv, hd))
    v[:, 2] = rng.integers(1500, 2048, v[:, 2].shape)
    if chunks > 3:
        at[:, :, 3] = at[:, :, 2]
        v[:, 3] = -v[:, 2]
    k = torch.zeros((S, chunks, CHUNK, kv, hd), dtype=torch.float16)
    k[..., 0] = torch.from_numpy(at).permute(0, 2, 1)[:, :, None].half()
    q = torch.zeros((S, kv * group, hd), dtype=torch.float16)
    q[..., 0] = torch.from_numpy(size).reshape(-1).half()

    def pool(x):
        return x.reshape(-1, PAGE, kv, hd).half().cuda()

    pages = n // PAGE
    table = torch.arange(S * pages, dtype=torch.int32, device="cuda").view(S, pages)
    cache = capi.PagedKV(pool(k), pool(torch.from_numpy(v)), table)
    batch = capi.SeqBatch(torch.arange(S + 1, dtype=torch.int32, device="cuda"),
                          torch.full((S,), n, dtype=torch.int32, device="cuda"), S, 1, n)
    scale = float(np.float32(0.6931472))  # times fp32(log2 e) it is 1 in fp32: scores in powers of two
    assert np.float32(scale) * np.float32(1.4426950408889634) == 1
    out = torch.empty((S, kv * group, hd), dtype=torch.float16, device="cuda")
    if op == "paged":
        capi.attention_paged_f16(out, q.cuda(), batch, cache, scale)
    else:
        lists = torch.arange(pages, dtype=torch.int32, device="cuda").expand(S, kv, pages).contiguous()
        capi.attention_selected_f16(out, q.cuda(), lists, batch, cache, scale)

    score = (at[:, :, None, :] * size[None, :, :, None]).astype(np.float32)  # exact
    e = torch.exp2(torch.from_numpy(score - score.max(-1, keepdims=True)).cuda()).cpu().numpy()
    # (the weights of a chunk are 2^11: a power of two moves no rounding)
    parts = v.sum(2).transpose(0, 2, 1, 3)[:, :, None].astype(np.float32)
    want = joined(e, np.broadcast_to(parts, e.shape + (hd,)), np.float32(CHUNK), hd)
    got = out.cpu().numpy().reshape(want.shape)
    assert np.array_equal(got.view(np.uint16), want.view(np.uint16)), \
        (int((got != want).sum()), got.size, float(np.abs(got.astype(float) - want.astype(float)).max()))
