"""Attention over windows with first positions and over shared beginnings
(fo_paged_window_attention, fo_paged_prefix_attention) where numbers are at the
ends of their ranges, against the float64 forms and within the bounds of
test_gpu_reach.py unless a test says otherwise."""

import numpy as np
import pytest

import fo_cuda as F
import paged_reference as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_paged import Cache, dev, rows_of, within  # noqa: E402
from test_gpu_reach import SharedCache, attend, check_rows, prefix_case, seen_of, window_case  # noqa: E402


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


# Shared beginnings, by what computes them: the few rows' kernel both times; the many rows' for the beginning and the few
# rows' for the rest, of single rows and of more; the many rows' both times; each sequence over all it sees.
FORMS = {"few": (4, 1, 2, False), "many and few": (40, 1, 2, False), "many and few, rows": (4, 20, 1, False),
         "many": (4, 20, 1, True), "alone": (4, 70, 1, False)}


def positive_keys(cache):
    if cache.fmt == "i8":
        cache.codes[0] = np.abs(cache.codes[0].view(np.int8)).view(np.uint8)
    else:
        cache.codes[0] &= 0x7F


class SharedForm:
    """Sequences of one group over a beginning of 3 1/2 pages, the third shorter than it.  (`below`: all scores below 0.)"""

    def __init__(self, form, seed, fmt, dim, dtype, below=False):
        self.seqs, self.n, self.group, wide = FORMS[form]
        rng, page = np.random.default_rng(seed), 128 if wide else 16
        self.page, self.shared = page, 3 * page + page // 2
        lens = [self.shared + self.n + 9 * b % 40 for b in range(self.seqs)]
        lens[2] = page + page // 2 + self.n // 2
        self.cache = SharedCache(rng, fmt, dim, page, 1, lens, [0, self.seqs], [self.shared])
        if wide:  # more positions than the few rows' kernel takes with several rows
            table = np.full((self.seqs, 8192 // page + 1), -7, np.int32)
            table[:, :self.cache.table.shape[1]] = self.cache.table
            self.cache.table = table
        if below:
            positive_keys(self.cache)
        self.kv = self.cache.on_device()
        self.values = [(self.cache.values(0, b), self.cache.values(1, b)) for b in range(self.seqs)]
        self.q, _ = rows_of(rng, self.seqs * self.n, self.group, dim, dtype)
        if below:
            self.q = -self.q.abs()
        self.places = np.concatenate([np.arange(n - self.n, n) for n in lens])
        self.dtype, self.scale = dtype, dim ** -0.5

    def attend(self, scale=None, ctx=None):
        groups = F.PagedGroups(dev(np.array([0, self.seqs], np.int32)), dev(np.array([self.shared], np.int32)))
        out, lse = torch.full_like(self.q, 9.0), torch.full(self.q.shape[:2], 9.0, device="cuda")
        F.paged_prefix_attention(self.kv, self.cache.batch([self.n] * self.seqs, False), groups, self.q, out, lse=lse,
                                 scale=scale, ctx=ctx)
        return out, lse

    def check(self, out, lse, rows, scale=None):
        """The rows whose numbers are given against the float64 form."""
        check_rows(out, lse, self.q.double().cpu().numpy(), [self.n] * self.seqs, self.cache.lens,
                   lambda b: self.values[b], lambda p: seen_of(p, 0, 0), None, self.scale if scale is None else scale,
                   self.dtype, only={(int(r) // self.n, int(r) % self.n) for r in rows})


WHAT = ["number", "k inf", "k -inf", "k nan", "v inf", "v -inf", "v nan"]


def damage(cache, seq, page, what):
    """A page number outside the pool, or a scale that is not finite (on the device; the cache keeps what was there)."""
    if what == "number":
        cache.table[seq, page] = 1 << 30
    else:
        cache.dev[2 if what[0] == "k" else 3][int(cache.table[seq, page])] = float(what[2:])


@pytest.mark.parametrize("fmt,dim,dtype", [("i8", 64, "bf16"), ("e4m3", 128, "f32")])
@pytest.mark.parametrize("what", WHAT)
@pytest.mark.parametrize("rows", [1, 12, 20, 60])
def test_a_lost_page_in_windows(fmt, dim, dtype, what, rows):
    """Rows that see the page give NaN, scores below 0 or not, and the others what they give without it."""
    for n, window, first in ((70, 1000, 1), (120, 30, 50)):
        rng = np.random.default_rng(4)
        cache = Cache(rng, fmt, dim, 16, 1, [n])
        positive_keys(cache)
        values, kv = [cache.values(i, 0) for i in range(2)], cache.on_device()
        damage(cache, 0, 3, what)
        q, _ = rows_of(rng, rows, 2, dim, dtype)
        q = -q.abs()
        ctx = F.Context(0)
        out, lse = torch.full_like(q, 9.0), torch.full((rows, 2), 9.0, device="cuda")
        F.paged_window_attention(kv, cache.batch([rows], False), q, out, window=window, first=first, lse=lse, ctx=ctx)
        sees = np.arange(n - rows, n) >= 48  # by the first positions, or a window longer than the sequence
        if what == "number":
            with pytest.raises(F.FoError, match="page table"):
                ctx.synchronize()
        ctx.synchronize()
        ctx.close()
        assert out[torch.from_numpy(sees).cuda()].isnan().all() and lse[torch.from_numpy(sees).cuda()].isnan().all()
        check_rows(out, lse, q.double().cpu().numpy(), [rows], [n], lambda b: values, lambda p: seen_of(p, window, first),
                   None, dim ** -0.5, dtype, only={(0, int(r)) for r in np.nonzero(~sees)[0]})


@pytest.mark.parametrize("fmt,dim,dtype", [("i8", 64, "bf16"), ("e4m3", 128, "f32")])
@pytest.mark.parametrize("what", WHAT)
@pytest.mark.parametrize("call,rows,window,first", [("window", rows, *reach) for rows in (12, 20, 60)
                                                    for reach in ((0, 0), (20, 0), (0, 7), (20, 7))] + [("no groups", 12, 0, 0)])
def test_a_lost_page_whatever_the_window(fmt, dim, dtype, what, call, rows, window, first):
    """Rows before the page, and those whose window is behind it, with and without first positions."""
    rng, n = np.random.default_rng(6), 90
    cache = Cache(rng, fmt, dim, 16, 1, [n])
    values, kv = [cache.values(i, 0) for i in range(2)], cache.on_device()
    lost = (n - rows // 2) // 16  # the page that the rows come to half way
    damage(cache, 0, lost, what)
    q, _ = rows_of(rng, rows, 2, dim, dtype)
    out, lse, ctx = torch.full_like(q, 9.0), torch.full((rows, 2), 9.0, device="cuda"), F.Context(0)
    if call == "window":
        F.paged_window_attention(kv, cache.batch([rows], False), q, out, window=window, first=first, lse=lse, ctx=ctx)
    else:
        groups = F.PagedGroups(dev(np.array([0], np.int32)), torch.empty(0, dtype=torch.int32, device="cuda"))
        F.paged_prefix_attention(kv, cache.batch([rows], False), groups, q, out, lse=lse, ctx=ctx)
    if what == "number":
        with pytest.raises(F.FoError, match="page table"):
            ctx.synchronize()
    ctx.synchronize()
    ctx.close()
    place = np.arange(n - rows, n)
    sees = place >= 16 * lost
    if window:
        sees &= place - (16 * lost + 15) < window
    assert sees.any()
    others = {(0, int(r)) for r in np.nonzero(~sees)[0]}
    check_rows(out, lse, q.double().cpu().numpy(), [rows], [n], lambda b: values, lambda p: seen_of(p, window, first), None,
               dim ** -0.5, dtype, only=others)
    at = torch.from_numpy(sees).cuda()
    # (A key scale of infinity: some of a row's scores are above 0.)
    assert out[at].isnan().all() and lse[at].isnan().all()


@pytest.mark.parametrize("fmt,dim,dtype", [("i8", 64, "bf16"), ("e4m3", 128, "f32")])
@pytest.mark.parametrize("what", WHAT)
@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("where", ["beginning", "behind one", "own"])
def test_a_lost_page_of_shared_beginnings(form, where, what, fmt, dim, dtype):
    """Of the beginning: lost to the rows of all sequences that come to it (one ends before its third page).  Of one
    sequence's own: to its rows alone."""
    f = SharedForm(form, 5, fmt, dim, dtype, below=True)
    seq, page = {"beginning": (0, 1), "behind one": (0, 2), "own": (1, f.shared // f.page)}[where]
    damage(f.cache, seq, page, what)
    ctx = F.Context(0)
    out, lse = f.attend(ctx=ctx)
    if what == "number":
        with pytest.raises(F.FoError, match="page table"):
            ctx.synchronize()
    ctx.synchronize()
    ctx.close()
    sees = f.places >= page * f.page
    if where == "own":
        sees = (np.arange(len(f.places)) // f.n == 1) & (f.places >= f.shared)
    assert sees.any()
    at = torch.from_numpy(sees).cuda()
    assert out[at].isnan().all() and lse[at].isnan().all()
    f.check(out, lse, np.nonzero(~sees)[0])



@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("scale", [None, -0.3, 0.0, 1e-3])
def test_queries_of_shared_beginnings(form, dtype, scale):
    """Rows of zeros, tiny and large ones beside ordinary ones; rows that are not finite are NaN and alone."""
    for fmt, dim in (("i8", 64), ("e4m3", 128)):
        f = SharedForm(form, 10, fmt, dim, dtype)
        total = len(f.places)
        f.q[0::4] = 0
        f.q[1::4] *= 1e-30
        f.q[2::4] *= 8
        out, lse = f.attend(scale)
        f.check(out, lse, range(0, total, max(total // 40, 1)), scale)
        bad = [1, 2, total - 1] if total > 4 else [1, 2]
        f.q[bad[0]], f.q[bad[1], 0, 3], f.q[bad[-1], -1, 9] = np.nan, np.inf, -np.inf
        again, lse_again = f.attend(scale)
        heads = torch.ones(total, f.group, dtype=torch.bool, device="cuda")
        heads[bad[0]], heads[bad[1], 0], heads[bad[-1], -1] = False, False, False
        assert torch.equal(again[heads], out[heads]) and torch.equal(lse_again[heads], lse[heads])
        assert again[~heads].isnan().all() and lse_again[~heads].isnan().all()


# ------------------------------------------------ both sides of the kernels' limits
@pytest.mark.parametrize("rows", [20, 60])
@pytest.mark.parametrize("dim", [64, 128])
def test_scales_of_queries_in_every_kernel(rows, dim):
    """Two query heads: 40 rows of a KV head of 64 are the few rows' kernel's, of 128, and 120, the many rows'."""
    window_case(7, "i8", dim, 32, 2, 2, "f32", [500], [rows], q_scale=1e-6, scale=1e5)
    window_case(7, "i8", dim, 32, 2, 2, "bf16", [500], [rows], q_scale=2.0 ** 20, scale=2.0 ** -21)
    window_case(8, "e4m3", dim, 32, 2, 2, "f32", [500], [rows], scale=3.0)
    for dtype in ("f32", "bf16"):
        window_case(9, "i8", dim, 32, 2, 2, dtype, [70], [rows], q_scale=0.0, window=30, first=3)
        window_case(9, "e4m3", dim, 32, 2, 2, dtype, [70], [rows], scale=-0.3, window=30, first=3)
        window_case(9, "i8", dim, 32, 2, 2, dtype, [300], [rows], scale=0.0)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_prompt_at_once_and_in_short_pieces(fmt, dtype):
    """The many rows' kernel for 120 rows, and the few rows' for the same in calls of 12: each is within its bound of
    the float64 form, so they are within twice that of each other."""
    rng = np.random.default_rng(11)
    n, rows, piece = 700, 120, 12
    for dim, window, first in ((64, 0, 0), (64, 100, 20), (128, 100, 20)):
        cache = Cache(rng, fmt, dim, 32, 2, [n])
        kv = cache.on_device()
        q, _ = rows_of(rng, rows, 4, dim, dtype)
        whole, lse = torch.full_like(q, 9.0), torch.full((rows, 4), 9.0, device="cuda")
        F.paged_window_attention(kv, cache.batch([rows], False), q, whole, window=window, first=first, lse=lse)
        pieces, lses = torch.full_like(q, 9.0), torch.full((rows, 4), 9.0, device="cuda")
        for r in range(0, rows, piece):
            batch = F.PagedBatch(dev(cache.table), dev(np.array([n - rows + r + piece], np.int32)), rows=piece)
            F.paged_window_attention(kv, batch, q[r:r + piece], pieces[r:r + piece], window=window, first=first,
                                     lse=lses[r:r + piece])
        values = [(cache.values(0, 0), cache.values(1, 0))]
        for out, z in ((whole, lse), (pieces, lses)):
            check_rows(out, z, q.double().cpu().numpy(), [rows], [n], lambda b: values[b],
                       lambda p: seen_of(p, window, first), None, dim ** -0.5, dtype)
        k, v = values[0]
        size = max(float((np.abs(k[h // 2]) @ np.abs(q[:, h].double().cpu().numpy().T)).max()) for h in range(4)) * dim ** -0.5
        d, top = 2.0 ** -17 * size, np.abs(v).max()
        bound = 2 * (4 * d + 2.0 ** -18 + (2.0 ** -11 if dtype == "bf16" else 2.0 ** -22)) * top
        if dtype == "bf16":
            bound += 2 * torch.finfo(torch.bfloat16).eps / 2 * top  # each rounded once
        assert float((whole.double() - pieces.double()).abs().max()) <= bound


@pytest.mark.parametrize("dim,dtype", [(64, "bf16"), (128, "f32")])
@pytest.mark.parametrize("prompt", [200, 900])
def test_a_decode_step_beside_a_prompt_over_shared_beginnings(dim, dtype, prompt):
    """Groups of several sequences, single rows beside prompts: below and above 64 query rows on average, in and out of
    groups."""
    rows = [1, 1, prompt, 1, 1, 0, 2, 1, 1, 70]
    own = [5, 40, prompt + 3, 1, 130, 2, 2, 9, 64, 90]
    some = {(b, r) for b, n in enumerate(rows) for r in range(n) if r < 3 or r % 61 == 0 or r == n - 1}
    prefix_case(12, "e4m3", dim, 32, 2, 2, dtype, [1, 5, 8], [333, 128], own, rows, ragged=True, only=some)
    prefix_case(13, "i8", dim, 16, 1, 4, dtype, [0, 10], [150], own, rows, ragged=True, only=some)


@pytest.mark.parametrize("group", [40, 100, 300])
@pytest.mark.parametrize("dim,dtype", [(64, "bf16"), (128, "f32")])
def test_many_query_heads(group, dim, dtype):
    """Units that end inside a row's heads, rows that are several units."""
    window_case(14, "i8", dim, 32, 1, group, dtype, [90, 3, 0, 200], [1] * 4, window=50, first=3)
    window_case(14, "e4m3", dim, 16, 2, group, dtype, [90, 40], [3, 0], ragged=True)
    prefix_case(15, "i8", dim, 32, 1, group, dtype, [0, 3], [100], [1, 30, 70], [1] * 3)
    prefix_case(15, "e4m3", dim, 16, 2, group, dtype, [0, 2, 3], [40, 16], [9, 30, 5], [2, 0, 5], ragged=True)


@pytest.mark.parametrize("form", list(FORMS))
def test_sinks_that_take_nothing_and_all(form):
    """Terms of 0 and of infinity; those of large sinks are exp(80)."""
    f = SharedForm(form, 16, "i8", 64, "f32")
    groups = F.PagedGroups(dev(np.array([0, f.seqs], np.int32)), dev(np.array([f.shared], np.int32)))
    batch, without = f.cache.batch([f.n] * f.seqs, False), f.attend()[0]
    for sink in (-np.inf, np.inf, 80.0):
        out, lse = torch.full_like(f.q, 9.0), torch.full(f.q.shape[:2], 9.0, device="cuda")
        F.paged_prefix_attention(f.kv, batch, groups, f.q, out, sinks=torch.full((f.group,), sink, device="cuda"), lse=lse)
        if sink == -np.inf:
            assert torch.equal(out, without)
        elif sink == np.inf:
            assert (out == 0).all()
        else:
            # out / without = e^lse / (e^lse + e^80): the exponent (some 116 in log2 units) is held to 2^-17, the
            # rest to 2^-18.
            expected = without.double() * (1 / (1 + torch.exp(80.0 - lse.double())))[..., None]
            assert ((out.double() - expected).abs() <= expected.abs() * (2.0 ** -16 + 2.0 ** -18)).all()
        assert lse[torch.from_numpy(f.places >= 0).cuda()].isfinite().all()


# ------------------------------------------------------------------ far positions, large pools
@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("rows", [1, 12, 60])
@pytest.mark.parametrize("first", [0, 20])
def test_windows_near_two_to_the_31(fmt, rows, first):
    """A table with room for nearly 2^31 positions whose pages between the first positions and the window are gone."""
    page, dim, window = 16, 64, 50
    room = (2 ** 31 - 1) // page
    n, near = room * page, 8 * page  # positions; those whose pages are there at the end
    rng = np.random.default_rng(20)
    cache = Cache(rng, fmt, dim, page, 2, [10 * page])
    table = torch.full((1, room), -1, dtype=torch.int32, device="cuda")
    table[0, :2] = dev(cache.table[0, :2])
    table[0, -8:] = dev(cache.table[0, 2:])
    kv = cache.on_device()
    q, _ = rows_of(rng, rows, 4, dim, "f32")
    out, lse, ctx = torch.full_like(q, 9.0), torch.full((rows, 4), 9.0, device="cuda"), F.Context(0)
    batch = F.PagedBatch(table, dev(np.array([n], np.int32)), rows=rows)
    F.paged_window_attention(kv, batch, q, out, window=window, first=first, lse=lse, ctx=ctx)
    ctx.synchronize()
    ctx.close()
    values = (cache.values(0, 0), cache.values(1, 0))

    def seen(p):  # of the pages that are there
        return np.concatenate((np.arange(first), np.arange(p + 1 - window, p + 1)))

    check_rows(out, lse, q.double().cpu().numpy(), [rows], [2 * page + near], lambda b: values, seen, None, dim ** -0.5, "f32")


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_offsets_beyond_32_bits(fmt):
    """The last pages of a pool of more than 2^32 bytes, by every kernel of the two calls."""
    page, kv_heads, dim, held = 128, 8, 128, 500
    pages = (1 << 32) // (page * kv_heads * dim) + 40
    rng = np.random.default_rng(21)
    small = Cache(rng, fmt, dim, page, kv_heads, [held])
    small.on_device()
    pool = [torch.zeros(pages, kv_heads, page, dim, dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.zeros(pages, kv_heads, device="cuda") for _ in range(2)]
    ids = np.arange(pages - 1, pages - 5, -1, dtype=np.int32)
    for i in range(2):
        for j, at in enumerate(ids):
            pool[i][int(at)] = small.dev[i][int(small.table[0, j])].view(torch.int8)
            scales[i][int(at)] = small.dev[2 + i][int(small.table[0, j])]
    kind = torch.int8 if fmt == "i8" else torch.float8_e4m3fn
    kv, values = F.PagedKv(*(c.view(kind) for c in pool), *scales), (small.values(0, 0), small.values(1, 0))
    for seqs, rows in ((1, 1), (40, 1), (2, 40), (1, 100)):  # (of shared beginnings, each in a form of its own)
        q, _ = rows_of(rng, seqs * rows, kv_heads, dim, "f32")
        batch = F.PagedBatch(dev(np.repeat(ids[None], seqs, 0)), dev(np.full(seqs, held, np.int32)), rows=rows)
        groups = F.PagedGroups(dev(np.array([0, seqs], np.int32)), dev(np.array([300], np.int32)))
        only = {(b, r) for b in range(0, seqs, 13) for r in range(0, rows, 9)}
        for call in ("window", "prefix"):
            out, lse = torch.full_like(q, 9.0), torch.full(q.shape[:2], 9.0, device="cuda")
            if call == "window":
                F.paged_window_attention(kv, batch, q, out, window=200, first=7, lse=lse)
            else:
                F.paged_prefix_attention(kv, batch, groups, q, out, lse=lse)
            check_rows(out, lse, q.double().cpu().numpy(), [rows] * seqs, [held] * seqs, lambda b: values,
                       lambda p: seen_of(p, 200, 7) if call == "window" else seen_of(p, 0, 0), None, dim ** -0.5, "f32", only)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("fmt,dim", [("i8", 64), ("e4m3", 128)])
@pytest.mark.parametrize("factor", [2.0 ** 20, 2.0 ** 24, 2.0 ** 30, 2.0 ** 60])
def test_scores_beyond_what_fp32_tells_apart(fmt, dim, dtype, factor):
    """Scores of 1e7 to 1e20, whose steps in FP32 are larger than a softmax's whole range: which positions win goes by
    rounding, and what comes out is a mean of values that the row sees (held to 2^-8 of the largest), never NaN."""
    rng = np.random.default_rng(22)
    cases = []
    for rows, window, first in ((4, 0, 0), (4, 60, 5), (100, 0, 0), (100, 60, 5), (300, 0, 0)):
        cache = Cache(rng, fmt, dim, 16, 1, [700, 320])
        q, _ = rows_of(rng, 2 * rows, 2, dim, dtype)
        q *= factor
        out, lse = attend_window(cache, [rows] * 2, q, window, first, 1.0)
        sequences = [(np.arange(n - rows, n), cache.values(1, b)) for b, n in enumerate(cache.lens)]
        cases.append((out, lse, sequences, window, first))
        if rows == 4:  # the older call's kernel is the same
            out, lse = torch.full_like(q, 9.0), torch.full(q.shape[:2], 9.0, device="cuda")
            F.paged_attention(cache.on_device(), cache.batch([rows] * 2, False), q, out, window=window, scale=1.0, lse=lse)
            cases.append((out, lse, sequences, window, 0))
    for form in FORMS:
        f = SharedForm(form, 23, fmt, dim, dtype)
        f.q *= factor
        out, lse = f.attend(1.0)
        cases.append((out, lse, [(f.places[b * f.n:(b + 1) * f.n], f.values[b][1]) for b in range(f.seqs)], 0, 0))
    for out, lse, sequences, window, first in cases:
        got, at = out.double().cpu().numpy(), 0
        for places, v in sequences:
            for p in places:
                seen = seen_of(int(p), window, first)
                top = np.abs(v[:, seen]).max(initial=0.0)
                assert (np.abs(got[at]) <= top * (1 + 2.0 ** -8)).all(), (p, got[at])
                at += 1
        assert not lse.isnan().any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("fmt,dim", [("i8", 64), ("e4m3", 128)])
@pytest.mark.parametrize("scale", [3e38, -3e38, 1e-30, 1e-40])
@pytest.mark.parametrize("keys", [1.0, 1e4])
def test_queries_of_zeros_at_any_scale(fmt, dim, dtype, scale, keys):
    """Scores of 0, whatever the scale argument and the keys' scales: the mean of what is in sight."""
    rng = np.random.default_rng(24)
    for rows, window, first in ((4, 60, 5), (100, 60, 5), (100, 0, 0)):
        cache = Cache(rng, fmt, dim, 16, 1, [300])
        cache.scales[0] *= np.float32(keys)
        q, _ = rows_of(rng, rows, 2, dim, dtype)
        q.zero_()
        out, lse = attend_window(cache, [rows], q, window, first, scale)
        check_rows(out, lse, q.double().cpu().numpy(), [rows], [300], lambda b: (cache.values(0, 0), cache.values(1, 0)),
                   lambda p: seen_of(p, window, first), None, scale, dtype)
    for form in FORMS:
        f = SharedForm(form, 25, fmt, dim, dtype)
        f.q.zero_()
        f.check(*f.attend(scale), range(0, len(f.places), max(len(f.places) // 30, 1)), scale)


# ------------------------------------------------------------------ the most there can be
@pytest.mark.parametrize("call", ["window", "window of few", "prefix", "prefix of one"])
def test_the_most_sequences(call):
    """65,535 of them, of 0 to 40 positions in pages that they share, some with many rows; as many groups."""
    rng = np.random.default_rng(26)
    n, page, dim = 65535, 16, 64
    cache = Cache(rng, "i8", dim, page, 1, [page] * 90)
    kv = cache.on_device()
    ids = cache.table[:, 0]
    table = ids[rng.integers(0, 90, (n, 3))].astype(np.int32)
    lens = rng.integers(0, 41, n).astype(np.int32)
    rows = np.minimum(1, lens) if call in ("window of few", "prefix") else np.where(rng.random(n) < 0.002, lens, np.minimum(lens, 1))
    start = np.concatenate(([0], np.cumsum(rows))).astype(np.int32)
    batch = F.PagedBatch(dev(table), dev(lens), rows=max(int(rows.max()), 1), row_start=dev(start))
    q, qv = rows_of(rng, int(start[-1]), 2, dim, "f32")
    out, lse, ctx = torch.full_like(q, 9.0), torch.full(q.shape[:2], 9.0, device="cuda"), F.Context(0)
    shared = np.zeros(n, np.int32)
    if call.startswith("window"):
        F.paged_window_attention(kv, batch, q, out, window=20, first=3, lse=lse, ctx=ctx)
    elif call == "prefix":  # every sequence a group of its own, over some of its positions
        shared = rng.integers(0, 41, n).astype(np.int32)
        groups = F.PagedGroups(dev(np.arange(n + 1, dtype=np.int32)), dev(shared))
        F.paged_prefix_attention(kv, batch, groups, q, out, lse=lse, ctx=ctx)
    else:  # one group of nearly all
        groups = F.PagedGroups(dev(np.array([1, n - 1], np.int32)), dev(np.array([page], np.int32)))
        table[1:n - 1, 0] = table[1, 0]
        F.paged_prefix_attention(kv, batch, groups, q, out, lse=lse, ctx=ctx)
    ctx.synchronize()
    ctx.close()
    got, got_lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    assert np.isfinite(got).all() and not np.isnan(got_lse).any()
    k, v = (R.decode(cache.codes[i], "i8") * cache.scales[i].astype(np.float64)[..., None, None] for i in range(2))
    some = set(rng.integers(0, n, 300).tolist()) | set(np.nonzero(rows > 1)[0].tolist()) | {0, 1, n - 2, n - 1}
    for b in sorted(some):
        kk, vv = (x[table[b]].transpose(1, 0, 2, 3).reshape(1, -1, dim)[:, :lens[b]] for x in (k, v))
        for r in range(rows[b]):
            at, p = start[b] + r, lens[b] - rows[b] + r
            seen = seen_of(int(p), 20, 3) if call.startswith("window") else seen_of(int(p), 0, 0)
            o, z, size, top = attend(qv[at], kk, vv, seen, None, dim ** -0.5)
            d = 2.0 ** -17 * size
            assert within(got[at], o, 4 * d * top + (2.0 ** -18 + 2.0 ** -22) * top, "f32")
            assert (np.abs(got_lse[at] - z) <= d + 2.0 ** -20 * (1 + np.abs(z))).all()


def test_a_beginning_of_a_sequence_without_positions():
    """The first of a group need only have the pages: its own length and rows may be none."""
    for form in ("few", "many and few", "many and few, rows", "many", "alone"):
        f = SharedForm(form, 27, "e4m3", 64, "bf16")
        lens, rows = list(f.cache.lens), [f.n] * f.seqs
        lens[0], rows[0] = 0, 0
        start = dev(np.concatenate(([0], np.cumsum(rows))).astype(np.int32))
        batch = F.PagedBatch(dev(f.cache.table), dev(np.array(lens, np.int32)), rows=f.n, row_start=start)
        groups = F.PagedGroups(dev(np.array([0, f.seqs], np.int32)), dev(np.array([f.shared], np.int32)))
        q = f.q[f.n:]
        out, lse, ctx = torch.full_like(q, 9.0), torch.full(q.shape[:2], 9.0, device="cuda"), F.Context(0)
        F.paged_prefix_attention(f.kv, batch, groups, q, out, lse=lse, ctx=ctx)
        ctx.synchronize()
        ctx.close()
        check_rows(out, lse, q.double().cpu().numpy(), rows, lens, lambda b: f.values[b], lambda p: seen_of(p, 0, 0), None,
                   0.125, "bf16", only={(b, r) for b in range(1, f.seqs) for r in range(0, f.n, 7)})
