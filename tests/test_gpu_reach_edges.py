"""Attention over windows with first positions and over shared beginnings
(fo_paged_window_attention, fo_paged_prefix_attention) where numbers are at the
ends of their ranges, against the float64 forms and within the bounds of
test_gpu_reach.py unless a test says otherwise."""

import numpy as np
import pytest

import fo_cuda as F

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_paged import Cache, dev, rows_of  # noqa: E402
from test_gpu_reach import check_rows, seen_of  # noqa: E402


def attend_window(cache, rows, q, window, first, scale=None, ctx=None):
    out, lse = torch.full_like(q, 9.0), torch.full(q.shape[:2], 9.0, device="cuda")
    F.paged_window_attention(cache.on_device(), cache.batch(rows, False), q, out, window=window, first=first, scale=scale,
                             lse=lse, ctx=ctx)
    return out, lse


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rows", [4, 100])
@pytest.mark.parametrize("key_scale,scale", [(1e-8, None), (3e-5, 1e-3), (1e-20, None)])
def test_small_keys_and_queries(dtype, dim, rows, key_scale, scale):
    """Queries of zeros, and tiny ones, over a page of tiny keys: what the mask leaves out stays out where the product
    of the scales is no longer above 0."""
    rng = np.random.default_rng(1)
    cache = Cache(rng, "i8", dim, 16, 1, [120, 131])
    for b in range(2):
        cache.scales[0][cache.table[b, 5]] = key_scale
        cache.scales[0][cache.table[b, 7]] = key_scale
    q, _ = rows_of(rng, 2 * rows, 2, dim, dtype)
    q[::3] = 0
    q[1::3, 1] *= 1e-30
    for window, first in ((0, 0), (30, 5)):
        out, lse = attend_window(cache, [rows] * 2, q, window, first, scale)
        check_rows(out, lse, q.double().cpu().numpy(), [rows] * 2, cache.lens,
                   lambda b: (cache.values(0, b), cache.values(1, b)), lambda p: seen_of(p, window, first), None,
                   dim ** -0.5 if scale is None else scale, dtype)
