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


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("call,rows,positions", [("prefix", 1, 16384), ("prefix", 1, 131072), ("prefix", 12, 131072),
                                                 ("window", 1, 131072), ("window", 60, 16384)])
def test_sums_of_long_sequences(fmt, dim, call, rows, positions):
    """FP32 rows over many positions of equal probability and values of one sign: what a sum loses at each step shows.

    Queries of zeros: scores are 0 and probabilities 1, without error.  A probability times its page's value scale is
    held to 2^-22, a step's own products and sums to 2^-21, the division and what joins parts to 2^-22.  Sums of steps
    are rounded to nearest, by 2^-24 of the total at most, as likely up as down: after n of them within 6 sqrt(n)
    2^-24 (six standard deviations at least), n being the positions by 64, a block of four warps with 16 a step.  Of
    many query rows n is the positions by 512, and the 64 additions between in the tensor core, which truncates,
    take 2^-23 each from what is there, half of the last sum on average."""
    seqs, heads, page = 40, 8, 64
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    n, pages = positions + page, positions // page + 1
    codes = torch.randint(64, 128, (2, pages, heads, page, dim), device="cuda", generator=g, dtype=torch.uint8)
    if fmt == "e4m3":
        codes = codes % 31 + 96  # 32 to 448
    codes = codes.view(torch.int8 if fmt == "i8" else torch.float8_e4m3fn)
    scales = torch.rand(2, pages, heads, device="cuda", generator=g) + 1.0
    kv = F.PagedKv(codes[0], codes[1], scales[0], scales[1])
    # (Every sequence reads the same pages.)
    table = torch.arange(pages, dtype=torch.int32, device="cuda").repeat(seqs, 1)
    batch = F.PagedBatch(table, torch.full((seqs,), n, dtype=torch.int32, device="cuda"), rows=rows)
    q = torch.zeros(seqs * rows, heads, dim, device="cuda")
    out = torch.empty_like(q)
    if call == "prefix":
        groups = F.PagedGroups(dev(np.array([0, seqs], np.int32)), dev(np.array([page], np.int32)))
        F.paged_prefix_attention(kv, batch, groups, q, out)
    else:
        F.paged_window_attention(kv, batch, q, out)
    total = torch.zeros(heads, dim, dtype=torch.float64, device="cuda")
    for i in range(0, pages, 256):
        x = codes[1, i:i + 256].to(torch.float64)
        total += (x.sum(2) * scales[1, i:i + 256, :, None].double()).sum(0)
    steps = positions / (512 if rows > 48 else 64)
    bound = 2.0 ** -22 + 2.0 ** -21 + 2.0 ** -22 + 6 * steps ** 0.5 * 2.0 ** -24 + (64 * 2.0 ** -23 / 2 if rows > 48 else 0)
    got = out.view(seqs, rows, heads, dim)[:, -1].double()  # the rows that see all
    assert float((got / (total / n) - 1).abs().max()) <= bound
