"""Rotary positions on several axes, attention over a window and first positions
that stay in sight, and attention of sequences that share their beginnings
(fo_rope_by_axes, fo_paged_append_by_axes, fo_paged_window_attention,
fo_paged_prefix_attention) against plain float64 implementations.

Bounds.  Rotations and appends as in test_gpu_paged.py: the same steps, so codes
and scales are compared for equality.  An attention's score s = scale * sum q k
is off by at most d = 2^-17 of the score's sum of magnitudes (FP32 sums of at
most 256 products, FP32 queries as two FP16 terms to 2^-22 of themselves), which
moves a probability by a factor e^d and the output by at most 4 d max|v|.  A
probability held as one FP16 is off by 2^-11 of itself (BF16 rows), as two by
2^-22 (FP32 rows): that share of max|v|, with FP32 sums, scales and divisions
2^-18 of max|v|; a probability below FP16's normal numbers, by 2^-35 of its
row's largest, of which there are fewer than 2^15.  max|v| is of the positions
that the row sees."""

import math

import numpy as np
import pytest

import fo_cuda as F
import paged_reference as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_paged import DTYPES, Cache, dev, plain_table, rows_of, within  # noqa: E402


def attend(q, k, v, seen, sinks, scale):
    """One row: q [heads][dim] over the positions `seen` of float64 k, v [kv heads][positions][dim]."""
    heads, kv_heads = q.shape[0], k.shape[0]
    out, lse, size = np.zeros(q.shape), np.full(heads, -np.inf), 0.0
    if len(seen) == 0:
        return out, lse, size, 0.0
    for h in range(heads):
        kk, vv = k[h // (heads // kv_heads)][seen], v[h // (heads // kv_heads)][seen]
        s = kk @ q[h] * scale
        size = max(size, float((np.abs(kk) @ np.abs(q[h])).max() * abs(scale)))
        m = s.max()
        p = np.exp(s - m)
        lse[h] = m + math.log(p.sum())
        out[h] = p @ vv / (p.sum() + (math.exp(sinks[h] - m) if sinks is not None else 0.0))
    return out, lse, size, float(np.abs(v[:, seen]).max())


def seen_of(position, window, first):
    if position < 0:
        return np.arange(0)
    low = max(0, position + 1 - window) if window else 0
    return np.concatenate((np.arange(min(first, low)), np.arange(low, position + 1)))


def check_rows(out, lse, qv, rows, lens, values, seen, sinks, scale, dtype, only=None):
    """Every row of out and lse against the float64 form; values(b) gives sequence b's keys and values."""
    got, got_lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    at = 0
    for b, n in enumerate(rows):
        k, v = values(b)
        for r in range(n):
            p = lens[b] - n + r
            if only is None or (b, r) in only:
                o, z, size, top = attend(qv[at], k, v, seen(p), sinks, scale)
                d = 2.0 ** -17 * size
                bound = 4 * d * top + (2.0 ** -18 + (2.0 ** -11 if dtype == "bf16" else 2.0 ** -22)) * top
                assert within(got[at], o, bound, dtype), (b, r, np.abs(got[at] - o).max(), bound)
                if p < 0:
                    assert np.isneginf(got_lse[at]).all() and (got[at] == 0).all()
                else:
                    assert (np.abs(got_lse[at] - z) <= d + 2.0 ** -20 * (1 + np.abs(z))).all()
            at += 1


def window_case(seed, fmt, dim, page, kv_heads, group, dtype, lens, rows, window=0, first=0, sinks=True, ragged=False,
                scale=None, q_scale=1.0, order="rows", pad=0, ctx=None, cache=None, only=None):
    rng = np.random.default_rng(seed)
    cache = cache or Cache(rng, fmt, dim, page, kv_heads, lens)
    kv, batch = cache.on_device(), cache.batch(rows, ragged)
    heads, total = kv_heads * group, sum(rows)
    q, _ = rows_of(rng, total, heads, dim, dtype, order, pad)
    q = (q * q_scale).to(q.dtype) if q_scale != 1.0 else q
    sk = rng.standard_normal(heads).astype(np.float32) if sinks else None
    out = torch.full((total, heads, dim), 9.0, dtype=q.dtype, device="cuda")
    lse = torch.full((total, heads), 9.0, device="cuda")
    F.paged_window_attention(kv, batch, q, out, window=window, first=first, sinks=None if sk is None else dev(sk),
                             scale=scale, lse=lse, ctx=ctx)
    (ctx or F.stream_context(0)).synchronize()
    check_rows(out, lse, q.double().cpu().numpy(), rows, lens, lambda b: (cache.values(0, b), cache.values(1, b)),
               lambda p: seen_of(p, window, first), sk, dim ** -0.5 if scale is None else scale, dtype, only)
    return out, lse


# --------------------------------------------------------------- many query rows
@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_prompts(fmt, dtype, dim, page):
    """Whole prompts and continued ones, units of one and of two query tiles, a row that sees nothing."""
    window_case(1, fmt, dim, page, 2, 2, dtype, [150, 300, 149, 20], [150] * 4)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rows", [17, 64, 65, 128, 129, 257])
def test_prompt_rows(dtype, dim, rows):
    window_case(2, "i8", dim, 32, 1, 1, dtype, [rows, rows + 131, rows - 1], [rows] * 3)


@pytest.mark.parametrize("group", [1, 3, 5, 8, 16])
def test_prompt_groups_of_heads(group):
    window_case(3, "e4m3", 64, 16, 2, group, "bf16", [70, 200], [70, 33], ragged=True)
    window_case(3, "i8", 128, 64, 2, group, "f32", [70, 200], [33, 40], ragged=True, sinks=False)


@pytest.mark.parametrize("window,first", [(1, 0), (1, 1), (2, 130), (64, 4), (100, 16), (127, 128), (128, 300), (129, 1),
                                          (300, 0), (5000, 7), (0, 9)])
@pytest.mark.parametrize("dim", [64, 128])
def test_prompt_windows(window, first, dim):
    window_case(4, "i8", dim, 16, 2, 2, "bf16", [400, 700], [400, 90], window=window, first=first, ragged=True)
    window_case(4, "e4m3", dim, 128, 1, 4, "f32", [333], [60], window=window, first=first)


@pytest.mark.parametrize("dim,dtype", [(64, "bf16"), (64, "f32"), (128, "bf16"), (128, "f32")])
def test_long_prompts_beside_short_ones(dim, dtype):
    """Sequences of more units than four, of few, of one row and of none in one batch; more units than threads."""
    lens = [1300, 5, 0, 1900, 700, 1, 0, 300, 2600, 9]
    rows = [1300, 1, 0, 1400, 700, 1, 0, 1, 1301, 9]
    rng = np.random.default_rng(26)
    some = {(b, int(r)) for b, n in enumerate(rows) if n for r in {0, n - 1, *rng.integers(0, n, 12), *range(127, n, 384)}}
    window_case(26, "i8", dim, 64, 1, 2, dtype, lens, rows, window=200, first=70, ragged=True, only=some)
    many = [3] * 500 + [1200] + [2] * 40
    some = {(b, r) for b in (0, 1, 250, 499, 501, 540) for r in (0, 1)} | {(500, r) for r in (0, 600, 1199)}
    window_case(27, "e4m3", dim, 16, 1, 1, dtype, many, many, window=30, first=2, ragged=True, only=some)


@pytest.mark.parametrize("group", [1, 2, 8, 16])
@pytest.mark.parametrize("fmt,dim,dtype", [("i8", 64, "bf16"), ("e4m3", 128, "f32"), ("e4m3", 64, "bf16"), ("i8", 128, "bf16")])
@pytest.mark.parametrize("window,first", [(90, 17), (0, 0), (60, 0), (1, 1)])
def test_a_decode_step_beside_prompts(group, fmt, dim, dtype, window, first):
    """Sequences of few rows go to one kernel and the others to the other: every row is written by one of them."""
    rows = [1, 1, 200, 1, 0, 1, 4, 1, 5, 8, 9, 1, 130, 1, 1, 2, 1, 0]
    lens = [1, 700, 200, 40, 0, 130, 90, 300, 3, 8, 500, 17, 333, 64, 65, 1, 999, 5]
    some = {(b, r) for b, n in enumerate(rows) for r in range(n) if r < 9 or r % 31 == 0 or r == n - 1}
    window_case(29, fmt, dim, 32, 1, group, dtype, lens, rows, window=window, first=first, ragged=True, only=some)


@pytest.mark.parametrize("dim,dtype", [(64, "bf16"), (128, "bf16"), (64, "f32"), (128, "f32")])
@pytest.mark.parametrize("long", [40, 700])
def test_shared_beginnings_of_a_decode_step_beside_prompts(dim, dtype, long):
    """Few rows on average and many at most: long prompts of several units beside single rows, in and out of groups."""
    rows = [1] * 14 + [long, 1, 0, 5] + [1] * 30 + [long // 2]
    own = [40 + 13 * (b % 5) + n for b, n in enumerate(rows)]
    some = {(b, r) for b, n in enumerate(rows) for r in range(n) if r < 2 or r % 97 == 0 or r == n - 1}
    prefix_case(30, "i8", dim, 32, 1, 2, dtype, [2, 12, 30, 30, 44], [333, 200, 0, 64], own, rows, ragged=True, only=some)


@pytest.mark.parametrize("dim,dtype", [(64, "bf16"), (128, "bf16"), (64, "f32"), (128, "f32")])
@pytest.mark.parametrize("ragged", [False, True])
def test_shared_beginnings_of_many_sequences_with_several_rows(dim, dtype, ragged):
    """20 query rows of a sequence: more sequences than one kernel takes, and as many as it does."""
    for fmt, seqs in (("i8", 110), ("e4m3", 7)):
        rows = [5 - b % 3 * ragged for b in range(seqs)]
        own = [n + 11 * b % 70 for b, n in enumerate(rows)]
        some = {(b, r) for b in range(0, seqs, 7) for r in range(rows[b])}
        prefix_case(31, fmt, dim, 16, 2, 4, dtype, [0, 3, seqs - 2], [100, 140], own, rows, ragged=ragged, only=some)


def test_rows_out_of_order_are_reported():
    """Of long prompts: the sequence whose rows end before they begin, and nothing else, is left out."""
    rng = np.random.default_rng(28)
    cache = Cache(rng, "i8", 64, 16, 1, [2000, 50, 110])
    start = dev(np.array([0, 2000, 1990, 2100], np.int32))
    batch = F.PagedBatch(dev(cache.table), dev(np.array(cache.lens, np.int32)), rows=2000, row_start=start)
    q, _ = rows_of(rng, 2100, 1, 64, "bf16")
    out = torch.empty_like(q)
    ctx = F.Context(0)
    F.paged_window_attention(cache.on_device(), batch, q, out, window=100, first=1, ctx=ctx)
    with pytest.raises(F.FoError, match="page table"):
        ctx.synchronize()
    ctx.synchronize()
    ctx.close()


@pytest.mark.parametrize("dim,group,rows", [(64, 8, 3), (64, 5, 8), (64, 8, 6), (64, 7, 7), (128, 6, 4), (128, 5, 5)])
@pytest.mark.parametrize("fmt,dtype", [("i8", "bf16"), ("e4m3", "f32")])
def test_rows_on_both_sides_of_the_kernels_limits(dim, group, rows, fmt, dtype):
    """24, 40, 48 and 49 query rows of a KV head; 24 and 25."""
    lens = [1, rows, rows + 1, 130, 257, 700]
    window_case(18, fmt, dim, 32, 2, group, dtype, lens, [min(n, rows) for n in lens], window=90, first=17, ragged=True)


@pytest.mark.parametrize("rows", [1, 60])
@pytest.mark.parametrize("first", [1000, 2 ** 31 - 1, 2 ** 40])
def test_more_first_positions_than_there_are(rows, first):
    """Nothing wraps, and what lies before the window stays in sight."""
    for fmt, dim, page in (("e4m3", 64, 128), ("e4m3", 128, 16), ("i8", 64, 64)):
        window_case(19, fmt, dim, page, 2, 2, "bf16", [100, 400, 999], [rows] * 3, window=50, first=first)


@pytest.mark.parametrize("window,first", [(1, 0), (1, 1), (2, 130), (64, 4), (100, 16), (200, 65), (5000, 7), (0, 9)])
@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("page", [16, 64, 128])
def test_few_rows_windows(window, first, fmt, page):
    lens = [0, 1, 64, 129, 700, 301]
    window_case(5, fmt, 64, page, 2, 2, "bf16", lens, [1] * 6, window=window, first=first)
    window_case(6, fmt, 128, page, 2, 2, "f32", lens, [4] * 6, window=window, first=first)


def test_ragged_orders_and_padding():
    lens, rows = [500, 90, 3, 1200, 7, 0], [101, 5, 0, 33, 7, 20]
    for order in ("rows", "heads"):
        window_case(7, "i8", 128, 32, 2, 4, "bf16", lens, rows, ragged=True, order=order, pad=5, window=100, first=3)
        window_case(7, "e4m3", 64, 16, 4, 2, "f32", lens, rows, ragged=True, order=order, pad=5)


def test_unaligned_rows():
    """Queries and outputs off 16-byte boundaries."""
    rng = np.random.default_rng(8)
    cache = Cache(rng, "i8", 64, 32, 2, [200])
    flat = torch.from_numpy(rng.standard_normal(60 * 4 * 64 + 1).astype(np.float32)).bfloat16().cuda()
    q = flat[1:].view(60, 4, 64)
    room = torch.zeros(60 * 4 * 64 + 1, dtype=torch.bfloat16, device="cuda")
    out, lse = room[1:].view(60, 4, 64), torch.empty(60, 4, device="cuda")
    F.paged_window_attention(cache.on_device(), cache.batch([60], False), q, out, window=50, first=2, lse=lse)
    check_rows(out, lse, q.double().cpu().numpy(), [60], [200], lambda b: (cache.values(0, b), cache.values(1, b)),
               lambda p: seen_of(p, 50, 2), None, 0.125, "bf16")


def test_many_sequences_and_a_long_one():
    lens = [int(n) for n in np.random.default_rng(0).integers(0, 150, 600)]
    rows = [int(n) for n in np.random.default_rng(1).integers(0, 20, 600)]
    window_case(9, "i8", 64, 16, 2, 2, "bf16", lens, rows, ragged=True, window=40, first=4)
    only = {(0, r) for r in range(0, 3000, 331)} | {(0, 2999)}
    window_case(10, "e4m3", 64, 64, 8, 2, "bf16", [9001], [3000], window=700, first=70, only=only)
    window_case(11, "i8", 128, 128, 8, 4, "bf16", [5001], [3000], only=only)
    window_case(12, "i8", 64, 64, 8, 2, "f32", [5001], [3000], only=only)


def test_scales_of_queries():
    window_case(13, "i8", 64, 32, 2, 2, "f32", [500], [20], q_scale=1e-6, scale=1e5)
    window_case(13, "i8", 128, 32, 2, 2, "bf16", [500], [20], q_scale=2.0 ** 20, scale=2.0 ** -21)
    window_case(14, "e4m3", 64, 32, 2, 2, "f32", [500], [20], scale=3.0)
    window_case(15, "i8", 64, 32, 2, 2, "f32", [70], [20], q_scale=0.0)
    window_case(15, "i8", 64, 32, 2, 2, "bf16", [70], [20], scale=-0.3)
    window_case(15, "i8", 64, 32, 2, 2, "bf16", [300], [20], scale=0.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_pages_of_very_different_scales(dtype):
    """A page whose values are 2^40 times another's does not touch the rows that do not see it."""
    rng = np.random.default_rng(16)
    cache = Cache(rng, "i8", 64, 16, 1, [200])
    cache.scales[1][cache.table[0, 9]] *= 2.0 ** 40
    cache.scales[1][cache.table[0, 2]] *= 2.0 ** -40
    cache.scales[1][cache.table[0, 3]] = 0.0  # values of zero, whatever the codes
    cache.scales[0][cache.table[0, 1]] = 0.0  # a page of zero keys
    window_case(17, "i8", 64, 16, 1, 1, dtype, [200], [200], cache=cache)
    window_case(17, "i8", 64, 16, 1, 1, dtype, [200], [200], cache=cache, window=16, first=1)


def test_growing_scores():
    """Scores that rise along the sequence move every row's maximum many times."""
    rng = np.random.default_rng(18)
    cache = Cache(rng, "i8", 64, 16, 1, [700])
    for j in range(44):
        cache.scales[0][cache.table[0, j]] *= 1 + j
    for dtype in ("bf16", "f32"):
        window_case(19, "i8", 64, 16, 1, 2, dtype, [700], [80], cache=cache, only={(0, r) for r in range(0, 80, 9)})
        window_case(19, "i8", 64, 16, 1, 1, dtype, [700], [80], cache=cache, only={(0, r) for r in range(0, 80, 9)})


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_queries_that_are_not_finite(bad, dtype):
    rng = np.random.default_rng(20)
    cache = Cache(rng, "e4m3", 64, 16, 1, [40])
    q, _ = rows_of(rng, 44, 2, 64, dtype)
    q[2], q[30, 1, 5] = bad, bad  # a row that sees nothing, and one that does
    out, lse = torch.empty_like(q), torch.empty(44, 2, device="cuda")
    F.paged_window_attention(cache.on_device(), cache.batch([44], False), q, out, lse=lse)
    got = out.float().cpu().numpy()
    assert (got[:4] == 0).all() and torch.isneginf(lse[:4]).all()
    assert np.isnan(got[30, 1]).all() and np.isnan(float(lse[30, 1]))
    got[30, 1] = 0
    assert np.isfinite(got).all()


def test_rows_of_no_sequence_are_left_alone():
    rng = np.random.default_rng(21)
    cache = Cache(rng, "i8", 64, 16, 2, [100, 50])
    start = dev(np.array([3, 60, 93], np.int32))
    batch = F.PagedBatch(dev(cache.table), dev(np.array(cache.lens, np.int32)), rows=57, row_start=start)
    q, _ = rows_of(rng, 100, 2, 64, "bf16")
    groups = F.PagedGroups(dev(np.array([0, 2], np.int32)), dev(np.array([16], np.int32)))
    for call in ("window", "prefix"):
        out, lse = torch.full((100, 2, 64), 7.0, dtype=q.dtype, device="cuda"), torch.full((100, 2), 7.0, device="cuda")
        if call == "window":
            F.paged_window_attention(cache.on_device(), batch, q, out, lse=lse)
        else:
            F.paged_prefix_attention(cache.on_device(), batch, groups, q, out, lse=lse)
        for t in (out, lse):
            assert (t[:3] == 7).all() and (t[93:] == 7).all() and not (t[3:93] == 7).any()


def test_equal_results_between_runs_and_to_the_few_rows_kernel():
    a = window_case(22, "i8", 64, 64, 8, 2, "bf16", [2000, 300], [100, 100], only=set())
    b = window_case(22, "i8", 64, 64, 8, 2, "bf16", [2000, 300], [100, 100], only=set())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_older_pages_may_be_gone():
    """Page numbers that no row sees are not read."""
    rng = np.random.default_rng(23)
    for rows, page in ((1, 16), (40, 16), (40, 128)):
        cache = Cache(rng, "e4m3", 64, page, 1, [1000])
        keep = cache.table.copy()
        ids = np.arange(cache.table.shape[1])
        seen = (ids * page < 20) | ((ids + 1) * page > 1000 - rows + 1 - 100)
        values = [cache.values(i, 0) for i in range(2)]
        cache.table[0, ~seen] = -1
        q, _ = rows_of(rng, rows, 2, 64, "bf16")
        out, lse = torch.empty_like(q), torch.empty(rows, 2, device="cuda")
        ctx = F.Context(0)
        F.paged_window_attention(cache.on_device(), cache.batch([rows], False), q, out, window=100, first=20, lse=lse,
                                 ctx=ctx)
        ctx.synchronize()
        ctx.close()
        cache.table = keep
        check_rows(out, lse, q.double().cpu().numpy(), [rows], [1000], lambda b: values,
                   lambda p: seen_of(p, 100, 20), None, 0.125, "bf16")


def test_bad_tables_are_reported():
    rng = np.random.default_rng(24)
    for rows in (1, 40):
        cache = Cache(rng, "i8", 64, 16, 1, [60, 60])
        cache.table[1, 2] = 1 << 30
        q, _ = rows_of(rng, 2 * rows, 1, 64, "f32")
        out, lse = torch.empty_like(q), torch.empty(2 * rows, 1, device="cuda")
        ctx = F.Context(0)
        F.paged_window_attention(cache.on_device(), cache.batch([rows] * 2, False), q, out, window=1000, first=1, lse=lse,
                                 ctx=ctx)
        with pytest.raises(F.FoError, match="page table"):
            ctx.synchronize()
        ctx.synchronize()
        ctx.close()
        got = out.cpu().numpy()
        assert np.isfinite(got[:rows]).all()
        for r in range(rows):  # NaN where the page is in sight, and only there
            assert np.isnan(got[rows + r]).all() == (60 - rows + r >= 32)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("what", ["number", "k", "v"])
@pytest.mark.parametrize("rows", [24, 40, 60])
def test_a_bad_page_is_lost_to_the_rows_that_see_it_alone(fmt, what, rows):
    """A page number outside the pool, a key's scale of NaN, a value's that is infinite: the rows before that page, and those
    whose window is behind it, come out as without it."""
    for n, window, first in ((70, 1000, 1), (120, 30, 5)):
        rng = np.random.default_rng(25)
        cache = Cache(rng, fmt, 64, 16, 1, [n])
        values, page = [cache.values(i, 0) for i in range(2)], 3
        at = int(cache.table[0, page])
        kv = cache.on_device()
        if what == "number":
            cache.table[0, page] = 1 << 30
        else:
            cache.dev[2 if what == "k" else 3][at] = math.nan if what == "k" else math.inf
        q, _ = rows_of(rng, rows, 2, 64, "bf16")
        out, lse = torch.empty_like(q), torch.empty(rows, 2, device="cuda")
        ctx = F.Context(0)
        F.paged_window_attention(kv, cache.batch([rows], False), q, out, window=window, first=first, lse=lse, ctx=ctx)
        if what == "number" and n == 70:
            with pytest.raises(F.FoError, match="page table"):
                ctx.synchronize()
        torch.cuda.synchronize()
        ctx.close()
        place = np.arange(n - rows, n)
        sees = (place >= 48) & (place - 63 < window)
        assert sees.any() or n > 70
        assert not np.isfinite(out.float().cpu().numpy()[sees]).any()
        check_rows(out, lse, q.double().cpu().numpy(), [rows], [n], lambda b: values, lambda p: seen_of(p, window, first), None,
                   0.125, "bf16", only={(0, int(r)) for r in np.nonzero(~sees)[0]})


# -------------------------------------------------------------- shared beginnings
class SharedCache(Cache):
    """A cache whose groups of sequences have their first sequence's pages for the shared positions: of the page that
    a beginning ends in, the others hold garbage before their own positions."""

    def __init__(self, rng, fmt, dim, page, kv_heads, lens, starts, shared):
        super().__init__(rng, fmt, dim, page, kv_heads, lens)
        self.leader, self.shared = list(range(len(lens))), [0] * len(lens)
        for g, n in enumerate(shared):
            for b in range(starts[g], starts[g + 1]):
                self.leader[b], self.shared[b] = starts[g], n
        self.full = self.table.copy()
        for b in range(len(lens)):
            if self.leader[b] != b:
                n = self.shared[b]
                self.table[b, :n // page] = -9  # not read
                if n % page and n < lens[b]:
                    self.codes[0][self.table[b, n // page], :, :n % page] = 0x7F if fmt == "e4m3" else 0x55
                    self.codes[1][self.table[b, n // page], :, :n % page] = 0x7F if fmt == "e4m3" else 0x55

    def values(self, i, b):
        def own(b):
            n = self.lens[b]
            pages = self.full[b, :-(-n // self.page)]
            x = R.decode(self.codes[i][pages], self.fmt) * self.scales[i][pages].astype(np.float64)[..., None, None]
            return x.transpose(1, 0, 2, 3).reshape(x.shape[1], -1, x.shape[3])[:, :n]
        x, n = own(b).copy(), min(self.shared[b], self.lens[b])
        x[:, :n] = own(self.leader[b])[:, :n]
        return x


def prefix_case(seed, fmt, dim, page, kv_heads, group, dtype, starts, shared, own, rows, sinks=True, ragged=False,
                ctx=None, only=None, order="rows", pad=0):
    """own: each sequence's positions behind its group's beginning (its rows among them); a negative one leaves it
    short of the beginning."""
    rng = np.random.default_rng(seed)
    before = [0] * len(rows)
    for g, n in enumerate(shared):
        for b in range(starts[g], starts[g + 1]):
            before[b] = n
    lens = [max(p + n, 0) for p, n in zip(before, own)]
    for g, n in enumerate(shared):
        assert starts[g] == starts[g + 1] or lens[starts[g]] >= n  # the first sequence holds the beginning
    cache = SharedCache(rng, fmt, dim, page, kv_heads, lens, starts, shared)
    kv, batch = cache.on_device(), cache.batch(rows, ragged)
    groups = F.PagedGroups(dev(np.array(starts, np.int32)), dev(np.array(shared, np.int32)))
    heads, total = kv_heads * group, sum(rows)
    q, _ = rows_of(rng, total, heads, dim, dtype, order, pad)
    sk = rng.standard_normal(heads).astype(np.float32) if sinks else None
    out = torch.full((total, heads, dim), 9.0, dtype=q.dtype, device="cuda")
    lse = torch.full((total, heads), 9.0, device="cuda")
    F.paged_prefix_attention(kv, batch, groups, q, out, sinks=None if sk is None else dev(sk), lse=lse, ctx=ctx)
    (ctx or F.stream_context(0)).synchronize()
    check_rows(out, lse, q.double().cpu().numpy(), rows, lens, lambda b: (cache.values(0, b), cache.values(1, b)),
               lambda p: seen_of(p, 0, 0), sk, dim ** -0.5, dtype, only)
    return out, lse


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_shared_beginnings(fmt, dtype, dim, page):
    """Few sequences (one kernel) and many (the other), beginnings that end in a page, at its end, and none."""
    prefix_case(30, fmt, dim, page, 2, 2, dtype, [0, 3, 5], [200, 128], [1, 40, 130, 17, 3], [1] * 5)
    prefix_case(31, fmt, dim, page, 1, 4, dtype, [0, 20, 41], [300, 77], [1 + 7 * i % 90 for i in range(41)], [1] * 41)


@pytest.mark.parametrize("rows", [1, 2, 5, 8, 16, 40])
@pytest.mark.parametrize("group", [1, 2, 5, 8])
def test_shared_beginnings_rows(rows, group):
    """Rows of a sequence across the rules' borders, some before the beginning's end, one that sees nothing."""
    own = [rows + 3, rows, rows - 1, -150, rows + 200, rows + 1]
    prefix_case(32, "i8", 64, 16, 2, group, "bf16", [0, 6], [150], own, [rows] * 6)
    prefix_case(33, "e4m3", 128, 64, 1, group, "f32", [0, 6], [150], own, [rows] * 6, sinks=False)


def test_shared_beginnings_groups():
    """Sequences of no group before and behind the groups, a group without sequences, ragged rows, other orders."""
    own = [30, 70, 5, 9, 64, 8, 3, 33, 90]
    for rows in ([1, 2, 5, 0, 3, 4, 1, 1, 2], [30, 2, 5, 0, 40, 8, 1, 33, 20]):
        for order in ("rows", "heads"):
            prefix_case(34, "i8", 64, 32, 2, 2, "bf16", [1, 4, 4, 7], [90, 50, 128], own, rows, ragged=True, order=order,
                        pad=3)
            prefix_case(35, "e4m3", 128, 16, 2, 2, "f32", [2, 3, 9], [17, 33], own, rows, ragged=True, order=order)


def test_shared_beginnings_long():
    only = {(b, 0) for b in range(0, 64, 7)}
    own = [1 + 37 * i % 600 for i in range(64)]
    prefix_case(36, "e4m3", 64, 64, 8, 2, "bf16", [0, 64], [9000], own, [1] * 64, only=only)
    prefix_case(37, "i8", 128, 128, 2, 4, "f32", [0, 30, 64], [5000, 3001], own, [1] * 64, only=only)


def test_shared_beginnings_no_groups_and_equal_runs():
    a = prefix_case(38, "i8", 64, 16, 1, 2, "bf16", [0], [], [100, 30], [2, 2])
    b = prefix_case(39, "i8", 64, 16, 8, 2, "bf16", [0, 40], [1000], [5 + i for i in range(40)], [3] * 40, only=set())
    c = prefix_case(39, "i8", 64, 16, 8, 2, "bf16", [0, 40], [1000], [5 + i for i in range(40)], [3] * 40, only=set())
    assert a[0].isfinite().all() and torch.equal(b[0], c[0]) and torch.equal(b[1], c[1])


def test_bad_groups_are_reported():
    rng = np.random.default_rng(40)
    for seqs, starts, lens in ((4, [0, 5], [16]), (4, [2, 1], [16]), (4, [-1, 4], [16]), (4, [0, 4], [-2]),
                               (4, [0, 4], [1 << 30]), (40, [0, 41], [16]), (40, [0, 40], [1 << 30])):
        cache = Cache(rng, "i8", 64, 16, 1, [60] * seqs)
        for rows in (1, 5):
            q, _ = rows_of(rng, seqs * rows, 1, 64, "f32")
            out, ctx = torch.empty_like(q), F.Context(0)
            groups = F.PagedGroups(dev(np.array(starts, np.int32)), dev(np.array(lens, np.int32)))
            F.paged_prefix_attention(cache.on_device(), cache.batch([rows] * seqs, False), groups, q, out, ctx=ctx)
            with pytest.raises(F.FoError, match="do not fit"):
                ctx.synchronize()
            ctx.close()


# ------------------------------------------------------------ positions on axes
def axes_of(kind, pairs):
    return {"one": [0] * pairs, "sections": [0] * (pairs // 4) + [1] * (pairs // 4) + [2] * (pairs - pairs // 4 * 2),
            "turns": [i % 3 for i in range(pairs)], "four": [3 - i % 4 for i in range(pairs)],
            "last": [2] * pairs}[kind]


def gathered(table, axes, positions):
    """A table row of its own for every row: [rows][pairs][2]."""
    return np.stack([table[positions[a], i] for i, a in enumerate(axes)], 1)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["one", "sections", "turns", "four", "last"])
@pytest.mark.parametrize("rows,heads,dim,rot,order,pad,shift", [
    (1, 1, 64, 64, "rows", 0, 0), (7, 24, 64, 32, "rows", 8, 0), (33, 5, 128, 128, "heads", 0, 0),
    (19, 3, 128, 24, "rows", 1, 0), (6, 3, 66, 34, "rows", 0, 0), (5, 9, 64, 64, "rows", 0, 1),
    (70, 2, 256, 256, "rows", 0, 0)])
def test_rope_axes(layout, dtype, kind, rows, heads, dim, rot, order, pad, shift):
    rng = np.random.default_rng(rows * 1000 + dim + rot)
    x, xv = rows_of(rng, rows, heads, dim, dtype, order, pad)
    if shift:
        flat = torch.empty(x.numel() + shift, dtype=x.dtype, device="cuda")
        flat[shift:].view(x.shape).copy_(x)
        x = flat[shift:].view(x.shape)
    table, axes = plain_table(500, rot), axes_of(kind, rot // 2)
    positions = rng.integers(0, 500, (4, rows)).astype(np.int32)
    entries = gathered(table, axes, positions)
    rope = F.RopeAxes(dev(table), axes, layout)
    for inverse in (False, True):
        for where in (dev(positions), dev(positions.T).t()):  # axes before rows, and behind them
            expected = R.rotate(xv, entries, np.arange(rows), layout, inverse)
            out = torch.full((rows, heads, dim), 7.0, dtype=x.dtype, device="cuda")
            F.rope(x, out, rope, positions=where, inverse=inverse)
            got = out.double().cpu().numpy()
            bound = 3 * 2.0 ** -24 * R.rotate(np.abs(xv), np.abs(entries) * [1, -1], np.arange(rows), layout).max()
            assert within(got, expected, bound, dtype)
            assert np.array_equal(got[..., rot:], xv[..., rot:])
            own = x.clone(memory_format=torch.preserve_format)
            F.rope(own, own, rope, positions=where, inverse=inverse)
            assert torch.equal(own, out)


def test_text_on_all_axes_is_plain_rotation():
    rng = np.random.default_rng(50)
    x, _ = rows_of(rng, 40, 6, 64, "bf16")
    table, at = dev(plain_table(500, 64)), rng.integers(0, 500, 40).astype(np.int32)
    a = F.rope(x, torch.empty_like(x), F.RopeAxes(table, axes_of("turns", 32), "half"), dev(np.stack([at] * 3)))
    b = F.rope(x, torch.empty_like(x), F.Rope(table, "half"), dev(at))
    assert torch.equal(a, b)


def test_rope_axes_transpose_is_the_gradient():
    """<w, rope(x)> against central differences of a linear map (a step of 1/4: good to 1e-4), and the formula's."""
    rng = np.random.default_rng(51)
    x, w = rng.standard_normal((2, 3, 4, 64)).astype(np.float32)
    table, axes = plain_table(64, 32) * np.float32(1.25), axes_of("sections", 16)
    positions = rng.integers(0, 64, (3, 3)).astype(np.int32)
    for layout in ("interleaved", "half"):
        rope = F.RopeAxes(dev(table), axes, layout)
        g = F.rope(dev(w), torch.empty(3, 4, 64, device="cuda"), rope, dev(positions), inverse=True).cpu().numpy()
        assert np.abs(g - R.rotate(w.astype(np.float64), gathered(table, axes, positions), np.arange(3), layout,
                                   True)).max() < 1e-5

        def value(z):
            y = F.rope(dev(z), torch.empty(3, 4, 64, device="cuda"), rope, dev(positions))
            return float((y.double().cpu() * torch.from_numpy(w).double()).sum())

        for i in [(0, 0, 0), (0, 1, 17), (1, 3, 31), (2, 2, 16), (2, 0, 40), (1, 1, 1)]:
            up, down = x.copy(), x.copy()
            up[i] += 0.25
            down[i] -= 0.25
            assert abs((value(up) - value(down)) / 0.5 - g[i]) < 1e-4


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_rope_axes_outside_the_table(layout):
    """A position outside gives NaN to its axis's pairs alone; an axis that no pair has may stand anywhere."""
    ctx = F.Context(0)
    x, axes = torch.ones(4, 2, 64, device="cuda"), [0] * 8 + [2] * 8
    positions = dev(np.array([[9, 10, 3, 0], [-5, 1 << 30, 0, 0], [1, 2, -1, 9]], np.int32))
    out = F.rope(x, torch.zeros_like(x), F.RopeAxes(dev(plain_table(10, 32)), axes, layout), positions, ctx=ctx)
    with pytest.raises(F.FoError, match="outside its table"):
        ctx.synchronize()
    got = out.cpu().numpy()
    pair = np.arange(32) // 2 if layout == "interleaved" else np.arange(32) % 16
    for r, lost in enumerate([None, 0, 2, None]):
        expected = np.isin(pair, np.nonzero(np.array(axes) == lost)[0]) if lost is not None else np.zeros(32, bool)
        assert (np.isnan(got[r, :, :32]) == expected).all() and (got[r, :, 32:] == 1).all()
    F.rope(x[:1], torch.zeros_like(x[:1]), F.RopeAxes(dev(plain_table(10, 32)), axes, layout), positions[:, :1], ctx=ctx)
    ctx.synchronize()
    ctx.close()


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rows", [1, 5, 70])
@pytest.mark.parametrize("layout,rot", [("interleaved", 64), ("half", 64), ("half", 24), ("interleaved", 6)])
def test_append_axes(fmt, dtype, dim, rows, layout, rot):
    """Codes and scales bit for bit, and the queries beside them."""
    rng = np.random.default_rng(rows + dim + rot)
    held, heads, kv_heads = [0, 37, 64], 6, 3
    cache = Cache(rng, fmt, dim, 32, kv_heads, held, extra_positions=rows)
    cache.lens = [n + rows for n in held]
    total = 3 * rows
    k, kx = rows_of(rng, total, kv_heads, dim, dtype, pad=2)
    v, vx = rows_of(rng, total, kv_heads, dim, dtype, pad=2)
    q, qx = rows_of(rng, total, heads, dim, dtype)
    table, axes = plain_table(900, rot), axes_of("turns", rot // 2)
    positions = rng.integers(0, 900, (3, total)).astype(np.int32)
    entries = gathered(table, axes, positions)
    q_out = torch.full((total, heads, dim), 5.0, dtype=q.dtype, device="cuda")
    F.paged_append(cache.on_device(), cache.batch([rows] * 3, False), k, v, rope=F.RopeAxes(dev(table), axes, layout),
                   positions=dev(positions), q=q, q_out=q_out)
    kx = R.rotate(kx, entries, np.arange(total), layout, dtype=np.float32)
    R.append(cache.codes[0], cache.scales[0], kx, [rows] * 3, cache.lens, cache.table, fmt)
    R.append(cache.codes[1], cache.scales[1], vx.astype(np.float32), [rows] * 3, cache.lens, cache.table, fmt)
    cache.check()
    expected = torch.from_numpy(R.rotate(qx, entries, np.arange(total), layout, dtype=np.float32)).to(q.dtype)
    assert torch.equal(q_out.cpu(), expected)


# ------------------------------------------------------------------- together
def test_serving_steps_in_a_graph():
    """Readings of one page: the page's prompt appended on axes and attended in windows, then steps of append and
    attention over the shared beginning, replayed from a graph; against the same calls made one by one."""
    g = torch.Generator(device="cuda")
    g.manual_seed(60)
    seqs, prompt, steps, page, kv_heads, heads, dim = 6, 333, 4, 32, 2, 4, 64
    side = torch.cuda.Stream()
    outs = []
    for captured in (False, True):
        g.manual_seed(60)
        per = -(-(prompt + steps) // page)
        codes = [torch.zeros(seqs * per, kv_heads, page, dim, dtype=torch.int8, device="cuda") for _ in range(2)]
        scales = [torch.zeros(seqs * per, kv_heads, device="cuda") for _ in range(2)]
        kv = F.PagedKv(*codes, *scales)
        table = torch.arange(seqs * per, dtype=torch.int32, device="cuda").view(seqs, per)
        rope = F.RopeAxes(dev(plain_table(1000, dim)), axes_of("sections", dim // 2), "half")
        rows = torch.randn(prompt, heads + 2 * kv_heads, dim, device="cuda", generator=g).bfloat16()
        at = torch.arange(prompt, device="cuda", dtype=torch.int32)
        positions = torch.stack((at // 100, at // 10, at))
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.default_stream())
            lens = torch.tensor([prompt], dtype=torch.int32, device="cuda")
            one = F.PagedBatch(table[:1], lens, rows=prompt)
            q = torch.empty(prompt, heads, dim, dtype=torch.bfloat16, device="cuda")
            F.paged_append(kv, one, rows[:, heads:heads + kv_heads], rows[:, heads + kv_heads:], rope=rope,
                           positions=positions, q=rows[:, :heads], q_out=q)
            first = F.paged_window_attention(kv, one, q, torch.empty_like(q), window=64, first=4)
            # Every other reading begins with a copy of the page that the prompt ends in.
            for t in codes + scales:
                t[table[1:, prompt // page].long()] = t[table[0, prompt // page].long()].clone()
            lengths = torch.full((seqs,), prompt, dtype=torch.int32, device="cuda")
            batch = F.PagedBatch(table, lengths)
            groups = F.PagedGroups(torch.tensor([0, seqs], dtype=torch.int32, device="cuda"),
                                   torch.tensor([prompt], dtype=torch.int32, device="cuda"))
            new = torch.empty(seqs, heads + 2 * kv_heads, dim, dtype=torch.bfloat16, device="cuda")
            where = torch.empty(3, seqs, dtype=torch.int32, device="cuda")
            sq, out = (torch.empty(seqs, heads, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))

            def step():
                lengths.add_(1)
                where.copy_(lengths.expand(3, seqs))
                F.paged_append(kv, batch, new[:, heads:heads + kv_heads], new[:, heads + kv_heads:], rope=rope,
                               positions=where, q=new[:, :heads], q_out=sq)
                F.paged_prefix_attention(kv, batch, groups, sq, out)

            graph = None
            got = [first.clone()]
            for i in range(steps):
                new.copy_(torch.randn(new.shape, device="cuda", generator=g))
                if captured and graph is None:
                    graph = torch.cuda.CUDAGraph()
                    side.synchronize()
                    with torch.cuda.graph(graph, stream=side):
                        step()
                graph.replay() if graph else step()
                got.append(out.clone())
            F.stream_context(0).synchronize()
        outs.append(got)
    for a, b in zip(*outs):
        assert torch.equal(a, b) and a.isfinite().all()


def test_two_streams_at_once_and_a_graph_beside():
    """Each stream's context has scratch of its own: calls side by side, and a replayed graph of both kernels of a ragged
    batch, give what each gives alone."""
    rng = np.random.default_rng(62)
    rows = [1] * 12 + [600] + [1] * 4
    cache = Cache(rng, "e4m3", 64, 32, 2, [700 + 40 * b for b in range(17)])
    kv, batch = cache.on_device(), cache.batch(rows, True)
    step = cache.batch([3] * 17, False)
    groups = F.PagedGroups(dev(np.array([0, 9, 17], np.int32)), dev(np.array([600, 333], np.int32)))
    q, _ = rows_of(rng, sum(rows), 4, 64, "bf16")
    few, _ = rows_of(rng, 51, 4, 64, "bf16")
    window = lambda out: F.paged_window_attention(kv, batch, q, out, window=300, first=20)  # noqa: E731
    prefix = lambda out: F.paged_prefix_attention(kv, step, groups, few, out)  # noqa: E731
    streams = [torch.cuda.Stream() for _ in range(3)]
    expected = []
    for call, x in ((window, q), (prefix, few), (window, q)):
        with torch.cuda.stream(streams[len(expected)]):
            out = torch.empty_like(x)
            call(out)
            expected.append(out)
    torch.cuda.synchronize()
    assert torch.equal(expected[0], expected[2])
    graph, replayed = torch.cuda.CUDAGraph(), torch.empty_like(q)
    with torch.cuda.graph(graph, stream=streams[2]):
        window(replayed)
    outs = [torch.empty_like(q) for _ in range(20)], [torch.empty_like(few) for _ in range(20)]
    torch.cuda.synchronize()
    for i in range(20):
        with torch.cuda.stream(streams[0]):
            window(outs[0][i])
        with torch.cuda.stream(streams[1]):
            prefix(outs[1][i])
        with torch.cuda.stream(streams[2]):
            graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, expected[0]) for x in outs[0]) and all(torch.equal(x, expected[1]) for x in outs[1])
    assert torch.equal(replayed, expected[0])


def test_first_calls_inside_a_capture_are_refused():
    rng = np.random.default_rng(61)
    cache = Cache(rng, "i8", 64, 16, 1, [60] * 20)
    kv, batch = cache.on_device(), cache.batch([3] * 20, False)
    groups = F.PagedGroups(dev(np.array([0, 20], np.int32)), dev(np.array([32], np.int32)))
    q, _ = rows_of(rng, 60, 2, 64, "bf16")
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        F.paged_attention(kv, batch, q, out)  # the context and its first scratch
        side.synchronize()
        with pytest.raises(F.FoError, match="cannot be captured"):
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
                F.paged_prefix_attention(kv, batch, groups, q, out)
        F.paged_prefix_attention(kv, batch, groups, q, out)
        expected = out.clone()
        graph = torch.cuda.CUDAGraph()
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            F.paged_prefix_attention(kv, batch, groups, q, out)
        # A wider call makes larger scratch; the graph keeps its own.
        wide = Cache(rng, "i8", 64, 16, 1, [60] * 3000)
        many, _ = rows_of(rng, 9000, 2, 64, "bf16")
        F.paged_prefix_attention(wide.on_device(), wide.batch([3] * 3000, False), groups, many, torch.empty_like(many))
        out.zero_()
        graph.replay()
        side.synchronize()
        assert torch.equal(out, expected)


def test_calls_without_rows():
    kv = Cache(np.random.default_rng(62), "i8", 64, 16, 1, [16]).on_device()
    batch = F.PagedBatch(torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"),
                         rows=4, row_start=torch.zeros(2, dtype=torch.int32, device="cuda"))
    none = torch.empty(0, 2, 64, device="cuda")
    groups = F.PagedGroups(dev(np.array([0, 1], np.int32)), dev(np.array([3], np.int32)))
    F.paged_window_attention(kv, batch, none, none.clone(), window=3, first=1)
    F.paged_prefix_attention(kv, batch, groups, none, none.clone())
    rope = F.RopeAxes(dev(plain_table(10, 64)), [0] * 32)
    F.rope(none, none.clone(), rope, torch.zeros(1, 0, dtype=torch.int32, device="cuda"))
    F.stream_context(0).synchronize()
