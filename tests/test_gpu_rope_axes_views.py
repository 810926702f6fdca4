"""rxq4_qk_norm_rope_axes on views of coordinates: one row expanded over the axes, as text
has, rows apart, and a single axis."""
from __future__ import annotations

import pytest
import torch

import rxq4  # noqa: F401
from rxq4 import capi
from tests import serving_reference as ref
from tests.test_gpu_qk_rope import F16, freqs, inputs

pytestmark = pytest.mark.gpu


def run(new, lens, positions, axis_of):
    p = ref.Paged(31, 8, 2, 64, 16, new, lens)
    cache, batch = p.device(capi)
    q, k, v = (t.cuda() for t in inputs(p, F16, False, 32)[:3])
    out = torch.full((p.rows, 8, 64), 7.0, dtype=F16, device="cuda")
    capi.qk_norm_rope_axes(out, q, k, v, batch, cache, freqs(64).cuda(), positions, axis_of)
    return [t.cpu() for t in (out, *cache.tensors[:2])]


@pytest.mark.parametrize("new,lens", [([1], [40]), ([33, 5], [50, 9])])
@pytest.mark.parametrize("axes", [1, 3, 16])
def test_one_row_for_all_axes(new, lens, axes):
    n = sum(new)
    text = (torch.arange(n, dtype=torch.int32) * 7 - 3).cuda()
    axis_of = (torch.arange(32, dtype=torch.int32) % axes).cuda()
    whole = text[None].expand(axes, n).contiguous()
    want = run(new, lens, whole, axis_of)
    apart = torch.full((2 * axes, n + 9), -1, dtype=torch.int32, device="cuda")
    apart[::2, 4:4 + n] = whole
    for view in (text[None].expand(axes, n), apart[::2, 4:4 + n]):
        for a, b in zip(run(new, lens, view, axis_of), want):
            assert torch.equal(a, b)
