"""The rotary operators and the paged 8-bit KV cache on the GPU
(fo_rope_table, fo_rope, fo_paged_append, fo_paged_attention) against plain
float64 implementations (tests/paged_reference.py).

Bounds.  A rotation has two products and a sum, each rounded: 3 * 2^-24 of
|a c| + |b s|.  BF16 output lies between the roundings to BF16 of the exact
result less and plus the FP32 bound (rounding is monotonic).  An append's codes and scales are equal to the documented float32 steps.  An
attention's score s = scale * sum q k is off by at most d = 2^-17 of the score's
sum of magnitudes (FP32 sums of at most 128 products, queries held to 22 bits),
which moves a probability by a factor e^d and the output by at most 4 d max|v|;
FP32 probabilities, sums and divisions add 2^-18 max|v|; with BF16 rows the
probabilities carry 11 bits, 2^-11 max|v|."""

import math

import numpy as np
import pytest

import fo_cuda as F
import paged_reference as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def rows_of(rng, rows, heads, dim, dtype, order="rows", pad=0):
    """Random rows as (CUDA tensor in some order of memory, its float64 values)."""
    x = torch.from_numpy(rng.standard_normal((rows, heads + pad, dim)).astype(np.float32)).to(DTYPES[dtype])
    if order == "heads":  # heads before rows
        t = x.transpose(0, 1).contiguous().cuda().transpose(0, 1)[:, :heads]
    else:
        t = x.cuda()[:, :heads]
    return t, x[:, :heads].double().numpy()


def plain_table(positions, rot, theta=10000.0):
    f = theta ** (-2.0 * np.arange(rot // 2) / rot)
    a = np.arange(positions)[:, None] * f
    return np.stack((np.cos(a), np.sin(a)), -1).astype(np.float32)


def within(got, exact, bound, dtype):
    """Whether every value of `got` is a value within `bound` of the exact one, rounded to the type."""
    low, high = (torch.from_numpy(np.asarray(x)).to(torch.float64) for x in (exact - bound, exact + bound))
    if dtype == "bf16":
        low, high = low.to(torch.bfloat16).double(), high.to(torch.bfloat16).double()
    got = torch.from_numpy(got)
    return bool(((got >= low) & (got <= high)).all())


# ----------------------------------------------------------------- the table
@pytest.mark.parametrize("scaling", ["none", "linear", "ntk", "yarn"])
@pytest.mark.parametrize("rot", [2, 24, 64, 128])
def test_rope_table(scaling, rot):
    n, theta, factor, original = 70001, 10000.0, 4.0, 4096
    i = np.arange(rot // 2)
    f, m = theta ** (-2.0 * i / rot), 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "ntk" and rot > 2:
        f = (theta * factor ** (rot / (rot - 2))) ** (-2.0 * i / rot)
    elif scaling == "yarn":
        at = lambda turns: rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        low, high = max(math.floor(at(32)), 0), min(math.ceil(at(1)), rot - 1)
        ramp = np.clip((i - low) / max(high - low, 0.001), 0, 1)
        f, m = f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1
    a = np.arange(n)[:, None] * f
    expected = np.stack((np.cos(a), np.sin(a)), -1) * m
    table = torch.empty(n, rot // 2, 2, device="cuda")
    F.rope_table(table, theta, scaling, factor, original)
    got = table.cpu().numpy().astype(np.float64)
    # Half a unit of FP32, and FP64 angles off by some units of 70,000.
    assert np.abs(got - expected).max() <= 2.0 ** -24 * m + 1e-10


# -------------------------------------------------------------------- rotation
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,heads,dim,rot,order,pad,shift", [
    (1, 1, 64, 64, "rows", 0, 0),
    (7, 24, 64, 32, "rows", 8, 0),     # the temporal half, a part of wider rows
    (33, 5, 128, 128, "heads", 0, 0),  # heads before rows
    (19, 3, 128, 24, "rows", 1, 0),    # pairs that no group of eight divides
    (11, 2, 80, 80, "rows", 0, 0),
    (6, 3, 66, 34, "rows", 0, 0),      # a width that no group of eight divides
    (5, 9, 64, 64, "rows", 0, 1),      # off a 16-byte boundary
    (300, 40, 128, 64, "rows", 0, 0),
])
def test_rope(layout, dtype, rows, heads, dim, rot, order, pad, shift):
    rng = np.random.default_rng(rows * 1000 + dim + rot)
    x, xv = rows_of(rng, rows, heads, dim, dtype, order, pad)
    if shift:
        flat = torch.empty(x.numel() + shift, dtype=x.dtype, device="cuda")
        flat[shift:].view(x.shape).copy_(x)
        x = flat[shift:].view(x.shape)
    table = plain_table(500, rot)
    positions = rng.integers(0, 500, rows).astype(np.int32)
    rope = F.Rope(dev(table), layout)
    for inverse in (False, True):
        for where in (dev(positions), None):
            at = positions if where is not None else np.arange(rows)
            expected = R.rotate(xv, table, at, layout, inverse)
            out = torch.full((rows, heads, dim), 7.0, dtype=x.dtype, device="cuda")
            F.rope(x, out, rope, positions=where, inverse=inverse)
            got = out.double().cpu().numpy()
            bound = 3 * 2.0 ** -24 * R.rotate(np.abs(xv), np.abs(table) * [1, -1], at, layout).max()
            assert within(got, expected, bound, dtype)
            assert np.array_equal(got[..., rot:], xv[..., rot:])
            # In place the same bits.
            own = x.clone(memory_format=torch.preserve_format)
            F.rope(own, own, rope, positions=where, inverse=inverse)
            assert torch.equal(own, out)


def test_rope_transpose_is_the_gradient():
    """sum w * rope(x) changes by <transposed rotation of w, dx>: against central differences, which a linear map
    meets to rounding (FP32 values of some 10: differences over a step of 1/4 are good to 1e-4)."""
    rng = np.random.default_rng(5)
    x, w = rng.standard_normal((2, 3, 4, 64)).astype(np.float32)
    table = plain_table(64, 32) * np.float32(1.25)
    positions = dev(np.array([3, 60, 21], np.int32))
    for layout in ("interleaved", "half"):
        rope = F.Rope(dev(table), layout)
        g = F.rope(dev(w), torch.empty(3, 4, 64, device="cuda"), rope, positions, inverse=True).cpu().numpy()

        def value(z):
            y = F.rope(dev(z), torch.empty(3, 4, 64, device="cuda"), rope, positions)
            return float((y.double().cpu() * torch.from_numpy(w).double()).sum())

        for i in [(0, 0, 0), (0, 1, 17), (1, 3, 31), (2, 2, 16), (2, 0, 40), (1, 1, 1)]:
            up, down = x.copy(), x.copy()
            up[i] += 0.25
            down[i] -= 0.25
            assert abs((value(up) - value(down)) / 0.5 - g[i]) < 1e-4


def test_rope_position_outside_the_table():
    ctx = F.Context(0)
    x = torch.ones(3, 2, 64, device="cuda")
    out = torch.zeros_like(x)
    F.rope(x, out, F.Rope(dev(plain_table(10, 32))), dev(np.array([9, 10, -1], np.int32)), ctx=ctx)
    with pytest.raises(F.FoError, match="outside its table"):
        ctx.synchronize()
    ctx.synchronize()  # reported once
    got = out.cpu().numpy()
    assert np.isfinite(got[0]).all() and np.isnan(got[1:, :, :32]).all() and (got[1:, :, 32:] == 1).all()
    ctx.close()


# ----------------------------------------------------------------- paged cache
class Cache:
    """A pool with random contents, its pages handed out in any order; what no sequence holds is garbage (NaN codes
    and scales)."""

    def __init__(self, rng, fmt, dim, page, kv_heads, lens, spare=2, extra_positions=0):
        self.fmt, self.lens, self.page = fmt, list(lens), page
        per = [-(-(max(n, 0) + extra_positions) // page) for n in lens]
        width = max(max(per), 1)
        order = rng.permutation(sum(per) + spare)
        self.table = np.full((len(lens), width), -7, np.int32)  # what is not read may be anything
        at = 0
        for b, n in enumerate(per):
            self.table[b, :n] = order[at:at + n]
            at += n
        shape = (sum(per) + spare, kv_heads, page, dim)
        garbage = 0x7F if fmt == "e4m3" else 0x55
        self.codes = [np.full(shape, garbage, np.uint8) for _ in range(2)]
        self.scales = [np.full(shape[:2], np.nan, np.float32) for _ in range(2)]
        for b, n in enumerate(lens):
            for p in range(0, n, page):
                pg, m = self.table[b, p // page], min(page, n - p)
                for i in range(2):
                    x = rng.standard_normal((kv_heads, m, dim)).astype(np.float32)
                    scale = np.abs(x).max((1, 2)) / R.TOP[fmt] * rng.uniform(0.5, 2.0, kv_heads).astype(np.float32)
                    scale = np.maximum(scale, np.abs(x).max((1, 2)) / R.TOP[fmt]).astype(np.float32)
                    self.codes[i][pg, :, :m] = R.encode(np.clip(x / scale[:, None, None], -R.TOP[fmt], R.TOP[fmt]), fmt)
                    self.scales[i][pg] = scale

    def on_device(self):
        kind = torch.int8 if self.fmt == "i8" else torch.float8_e4m3fn
        self.dev = [dev(c).view(kind) for c in self.codes] + [dev(s) for s in self.scales]
        return F.PagedKv(*self.dev)

    def batch(self, rows, ragged):
        start = None
        if ragged:
            start = dev(np.concatenate(([0], np.cumsum(rows))).astype(np.int32))
        return F.PagedBatch(dev(self.table), dev(np.array(self.lens, np.int32)), rows=max(rows), row_start=start)

    def values(self, i, b):
        """float64 [kv heads][positions][dim] of sequence b's keys (0) or values (1)."""
        n = self.lens[b]
        pages = self.table[b, :-(-n // self.page)]
        x = R.decode(self.codes[i][pages], self.fmt) * self.scales[i][pages].astype(np.float64)[..., None, None]
        return x.transpose(1, 0, 2, 3).reshape(x.shape[1], -1, x.shape[3])[:, :n]

    def check(self, codes_equal_where=None):
        for i in range(2):
            got = self.dev[i].view(torch.uint8).cpu().numpy()
            assert np.array_equal(got, self.codes[i])
            assert np.array_equal(self.dev[2 + i].cpu().numpy().view(np.uint32), self.scales[i].view(np.uint32))


def attention_case(seed, fmt, dim, page, kv_heads, group, dtype, lens, rows, window=0, sinks=True, ragged=False,
                   scale=None, q_scale=1.0, order="rows", pad=0, ctx=None):
    rng = np.random.default_rng(seed)
    cache = Cache(rng, fmt, dim, page, kv_heads, lens)
    kv, batch = cache.on_device(), cache.batch(rows, ragged)
    heads, total = kv_heads * group, sum(rows)
    q, _ = rows_of(rng, total, heads, dim, dtype, order, pad)
    q = (q * q_scale).to(q.dtype) if q_scale != 1.0 else q
    qv = q.double().cpu().numpy()
    sk = rng.standard_normal(heads).astype(np.float32) if sinks else None
    out = torch.full((total, heads, dim), 9.0, dtype=q.dtype, device="cuda")
    lse = torch.full((total, heads), 9.0, device="cuda")
    F.paged_attention(kv, batch, q, out, sinks=None if sk is None else dev(sk), scale=scale, window=window, lse=lse,
                      ctx=ctx)
    got, got_lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    at = 0
    for b, n in enumerate(rows):
        k, v = cache.values(0, b), cache.values(1, b)
        top = np.abs(v).max(initial=0.0)
        for r in range(n):
            o, z, size = R.attend(qv[at], k, v, lens[b] - n + r, window, sk, dim ** -0.5 if scale is None else scale)
            d = 2.0 ** -17 * size
            bound = 4 * d * top + 2.0 ** -18 * top
            if dtype == "bf16":
                bound = bound + 2.0 ** -11 * top
            assert within(got[at], o, bound, dtype), (b, r, np.abs(got[at] - o).max(), bound)
            if lens[b] - n + r < 0:
                assert np.isneginf(got_lse[at]).all() and (got[at] == 0).all()
            else:
                assert (np.abs(got_lse[at] - z) <= d + 2.0 ** -20 * (1 + np.abs(z))).all()
            at += 1
    return out, lse


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_attention_lengths(fmt, dtype, dim, page):
    """One row each against lengths around every edge: none, one, a page's and a tile's end."""
    lens = [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 200, 777]
    attention_case(1, fmt, dim, page, 2, 2, dtype, lens, [1] * len(lens))


@pytest.mark.parametrize("group", [1, 2, 3, 5, 8, 16])
@pytest.mark.parametrize("rows", [1, 2, 5, 8])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_groups_and_rows(group, rows, dtype):
    lens = [300, rows - 1, rows, 70]  # the second has a row that sees nothing
    attention_case(2, "i8", 64, 32, 3, group, dtype, lens, [rows] * 4)
    attention_case(3, "e4m3", 128, 64, 1, group, dtype, lens, [rows] * 4, sinks=False)


@pytest.mark.parametrize("rows", [17, 64])
def test_attention_many_rows(rows):
    attention_case(4, "i8", 64, 16, 2, 4, "bf16", [400, 64], [rows] * 2)
    attention_case(4, "e4m3", 128, 16, 1, 4, "f32", [90], [rows])


@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 200, 5000])
def test_attention_window(window):
    lens = [1, 64, 129, 700]
    attention_case(5, "i8", 64, 16, 2, 4, "bf16", lens, [1] * 4, window=window)
    attention_case(6, "e4m3", 128, 32, 2, 2, "f32", lens, [4] * 4, window=window)


def test_attention_ragged_rows():
    attention_case(7, "i8", 128, 32, 2, 4, "bf16", [500, 90, 3, 1200, 7], [1, 5, 0, 3, 7], ragged=True)
    attention_case(7, "e4m3", 64, 16, 4, 2, "f32", [500, 90, 0, 2], [2, 0, 1, 8], ragged=True, window=100)


def test_attention_orders_of_memory():
    for order in ("rows", "heads"):
        attention_case(8, "i8", 64, 64, 2, 3, "bf16", [333, 40], [3, 3], order=order, pad=5)
        attention_case(8, "e4m3", 128, 64, 2, 3, "f32", [333, 40], [3, 3], order=order, pad=5)


def test_attention_one_long_sequence_and_many_short_ones():
    attention_case(9, "i8", 64, 64, 8, 2, "f32", [16384], [5])
    attention_case(9, "e4m3", 128, 128, 2, 4, "bf16", [9000, 1, 30, 5000], [1] * 4)
    lens = [int(n) for n in np.random.default_rng(0).integers(0, 150, 300)]
    attention_case(10, "i8", 64, 16, 2, 2, "bf16", lens, [1] * 300)


def test_attention_scales_of_queries():
    """Queries far from 1 (their magnitude must not matter to how they are held), and a peaked softmax."""
    attention_case(11, "i8", 64, 32, 2, 2, "f32", [500], [2], q_scale=1e-6, scale=1e5)
    attention_case(11, "i8", 128, 32, 2, 2, "bf16", [500], [2], q_scale=2.0 ** 20, scale=2.0 ** -21)
    attention_case(12, "e4m3", 64, 32, 2, 2, "f32", [500], [2], scale=3.0)
    attention_case(13, "i8", 64, 32, 2, 2, "f32", [70], [1], q_scale=0.0)
    attention_case(13, "i8", 64, 32, 2, 2, "bf16", [70], [1], scale=-0.3)


def test_attention_pages_of_very_different_scales():
    """A page whose values are 2^40 times another's: what it adds to small outputs is exact to its own size."""
    rng = np.random.default_rng(14)
    cache = Cache(rng, "i8", 64, 16, 1, [64])
    cache.scales[1][cache.table[0, 1]] *= 2.0 ** 40
    cache.scales[1][cache.table[0, 2]] *= 2.0 ** -40
    cache.scales[0][cache.table[0, 1]] = 0.0  # a page of zero keys
    kv, batch = cache.on_device(), cache.batch([1], False)
    q, qv = rows_of(rng, 1, 2, 64, "f32")
    out = torch.empty(1, 2, 64, device="cuda")
    F.paged_attention(kv, batch, q, out)
    k, v = cache.values(0, 0), cache.values(1, 0)
    o, _, _ = R.attend(qv[0], k, v, 63, 0, None, 0.125)
    got = out.double().cpu().numpy()[0]
    assert (np.abs(got - o) <= 2.0 ** -14 * np.abs(v).max()).all()
    # Without that page in sight, the others' accuracy is their own.
    F.paged_attention(kv, batch, q, out, window=32)
    o, _, _ = R.attend(qv[0], k, v, 63, 32, None, 0.125)
    assert (np.abs(out.double().cpu().numpy()[0] - o) <= 2.0 ** -14 * np.abs(v[:, 32:]).max()).all()


def test_attention_results_do_not_change_between_runs():
    a = attention_case(15, "i8", 64, 64, 8, 2, "bf16", [5000, 300, 8000], [1] * 3)
    b = attention_case(15, "i8", 64, 64, 8, 2, "bf16", [5000, 300, 8000], [1] * 3)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_attention_reports_bad_tables_and_lengths():
    rng = np.random.default_rng(16)
    cache = Cache(rng, "i8", 64, 16, 1, [40, 40])
    q, _ = rows_of(rng, 2, 1, 64, "f32")
    out = torch.empty(2, 1, 64, device="cuda")
    for change in ("page", "length"):
        ctx = F.Context(0)
        if change == "page":
            cache.table[1, 1] = 1 << 30
        else:
            cache.table[1, 1] = 0
            cache.lens[1] = 49  # a page more than its table has
        F.paged_attention(cache.on_device(), cache.batch([1, 1], False), q, out, ctx=ctx)
        with pytest.raises(F.FoError, match="page table"):
            ctx.synchronize()
        ctx.synchronize()
        o, _, _ = R.attend(q.double().cpu().numpy()[0], cache.values(0, 0), cache.values(1, 0), 39, 0, None, 0.125)
        assert np.abs(out.double().cpu().numpy()[0] - o).max() < 1e-4  # the other sequence is whole
        ctx.close()
    ctx = F.Context(0)
    cache.lens[1] = 40
    batch = F.PagedBatch(dev(cache.table), dev(np.array(cache.lens, np.int32)), rows=2,
                         row_start=dev(np.array([0, 1, 5], np.int32)))
    F.paged_attention(cache.on_device(), batch, q, out, ctx=ctx)
    with pytest.raises(F.FoError, match="row ranges"):
        ctx.synchronize()
    ctx.close()


# --------------------------------------------------------------------- append
def append_case(seed, fmt, dim, page, kv_heads, dtype, held, rows, layout="interleaved", rot=None, heads=0,
                ragged=False, order="rows", pad=0, positions=False, size=1.0):
    """Rows appended to sequences that hold `held` positions each."""
    rng = np.random.default_rng(seed)
    room = max(rows)
    cache = Cache(rng, fmt, dim, page, kv_heads, held, extra_positions=room)
    cache.lens = [n + m for n, m in zip(held, rows)]
    total = sum(rows)
    k, kx = rows_of(rng, total, kv_heads, dim, dtype, order, pad)
    v, vx = rows_of(rng, total, kv_heads, dim, dtype, order, pad)
    k, v = (k * size).to(k.dtype), (v * size).to(v.dtype)
    kx, vx = k.double().cpu().numpy(), v.double().cpu().numpy()
    kv, batch = cache.on_device(), cache.batch(rows, ragged)
    rope = where = q = q_out = None
    at = np.array([n + r for n, m in zip(held, rows) for r in range(m)])
    if rot:
        table = plain_table(4000, rot)
        rope = F.Rope(dev(table), layout)
        if positions:
            at = rng.integers(0, 4000, total)
            where = dev(at.astype(np.int32))
        if heads:
            q, qx = rows_of(rng, total, heads, dim, dtype, order, pad)
            q_out = torch.full((total, heads, dim), 5.0, dtype=q.dtype, device="cuda")
        kx = R.rotate(kx, table, at, layout, dtype=np.float32)
    F.paged_append(kv, batch, k, v, rope=rope, positions=where, q=q, q_out=q_out)
    R.append(cache.codes[0], cache.scales[0], kx.astype(np.float32), rows, cache.lens, cache.table, fmt)
    R.append(cache.codes[1], cache.scales[1], vx.astype(np.float32), rows, cache.lens, cache.table, fmt)
    cache.check()
    if heads:
        expected = torch.from_numpy(R.rotate(qx, table, at, layout, dtype=np.float32)).to(q.dtype)
        assert torch.equal(q_out.cpu(), expected)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_append_steps(fmt, dtype, dim, page):
    """Single rows and some at every place of a page, with scales that grow and that stay."""
    held = [0, 1, page - 1, page, page + 1, 3 * page - 2]
    for rows in (1, 3, 8):
        append_case(20, fmt, dim, page, 2, dtype, held, [rows] * 6, rot=dim, heads=4)
    append_case(21, fmt, dim, page, 2, dtype, held, [1] * 6, size=9.0)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 128])
def test_append_prompts(fmt, dtype, dim, page):
    append_case(22, fmt, dim, page, 3, dtype, [0, 5, page], [300] * 3, rot=dim // 2, layout="half", heads=6)
    append_case(23, fmt, dim, page, 1, dtype, [0, 7, 90, 0], [211, 1, 50, 0], rot=dim, heads=2, ragged=True, size=30.0)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("rot", [2, 24, 32, 64])
def test_append_rotations(layout, rot):
    for rows in (2, 40):
        append_case(24, "i8", 64, 32, 2, "f32", [10, 31], [rows] * 2, layout=layout, rot=rot, heads=3)
        append_case(25, "e4m3", 64, 32, 2, "bf16", [10, 31], [rows] * 2, layout=layout, rot=rot, heads=3,
                    positions=True, order="heads", pad=1)


def test_append_ragged_and_orders():
    append_case(26, "i8", 64, 16, 2, "bf16", [0, 9, 100, 3], [8, 0, 1, 5], ragged=True, rot=64, heads=2, pad=3)
    append_case(27, "e4m3", 128, 64, 2, "f32", [0, 9, 100, 3, 64], [500, 1, 2, 0, 129], ragged=True, rot=128, heads=2,
                order="heads")


def test_append_again_after_a_rejected_draft():
    """Lengths taken back and appended to again: the page keeps its (larger) scale, a page begun anew does not."""
    rng = np.random.default_rng(28)
    cache = Cache(rng, "i8", 64, 16, 1, [10], extra_positions=40)
    kv = cache.on_device()
    for n, m, size in [(20, 10, 50.0), (14, 4, 1.0), (17, 3, 1.0), (16, 1, 0.1), (18, 2, 0.01)]:
        cache.lens = [n]
        k, kx = rows_of(rng, m, 1, 64, "f32")
        k, kx = k * size, (k * size).cpu().numpy()
        F.paged_append(kv, cache.batch([m], False), k, k)
        R.append(cache.codes[0], cache.scales[0], kx, [m], cache.lens, cache.table, "i8")
        R.append(cache.codes[1], cache.scales[1], kx, [m], cache.lens, cache.table, "i8")
        cache.check()


def test_append_padded_slots_and_zeros():
    """Padded slots (length 0) store nothing; blocks of zeros have scale 0 and grow from it."""
    rng = np.random.default_rng(29)
    cache = Cache(rng, "e4m3", 64, 16, 1, [0, 3, 2], extra_positions=20)
    kv = cache.on_device()
    table = plain_table(50, 64)
    k = torch.zeros(3, 1, 64, device="cuda")
    k[2] = 4.0
    q, _ = rows_of(rng, 3, 2, 64, "f32")
    q_out = torch.empty_like(q)
    cache.lens = [0, 1, 3]
    ctx = F.Context(0)
    F.paged_append(kv, cache.batch([1] * 3, False), k, k, rope=F.Rope(dev(table)), q=q, q_out=q_out, ctx=ctx)
    ctx.synchronize()
    kx = R.rotate(k.cpu().numpy(), table, np.array([0, 0, 2]), "interleaved", dtype=np.float32)
    R.append(cache.codes[0], cache.scales[0], kx, [1] * 3, cache.lens, cache.table, "e4m3")
    R.append(cache.codes[1], cache.scales[1], k.cpu().numpy(), [1] * 3, cache.lens, cache.table, "e4m3")
    cache.check()
    assert cache.scales[0][cache.table[1, 0], 0] == 0
    assert torch.equal(q_out[0], q[0])
    ctx.close()


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("rows", [2, 40])
def test_append_values_that_are_not_finite(fmt, rows):
    rng = np.random.default_rng(30)
    cache = Cache(rng, fmt, 64, 32, 2, [5], extra_positions=rows)
    cache.lens = [5 + rows]
    kv = cache.on_device()
    k, kx = rows_of(rng, rows, 2, 64, "f32")
    k[0, 0, 3], k[1, 1, 9], k[1, 0, 7] = math.nan, math.inf, -math.inf
    ctx = F.Context(0)
    F.paged_append(kv, cache.batch([rows], False), k, k, ctx=ctx)
    with pytest.raises(F.NonFiniteError, match="not finite"):
        ctx.synchronize()
    ctx.synchronize()
    for i in range(2):
        R.append(cache.codes[i], cache.scales[i], k.cpu().numpy(), [rows], cache.lens, cache.table, fmt)
    cache.check()
    ctx.close()


def test_append_reports_bad_pages():
    rng = np.random.default_rng(31)
    cache = Cache(rng, "i8", 64, 16, 1, [3, 3], extra_positions=4)
    kv = cache.on_device()
    cache.lens = [4, 4]
    good = cache.table.copy()
    cache.table[1, 0] = -1
    ctx = F.Context(0)
    k, kx = rows_of(rng, 2, 1, 64, "f32")
    F.paged_append(kv, cache.batch([1, 1], False), k, k, ctx=ctx)
    with pytest.raises(F.FoError, match="page table"):
        ctx.synchronize()
    for i in range(2):
        R.append(cache.codes[i], cache.scales[i], kx.astype(np.float32)[:1], [1], [4], good[:1], "i8")
    cache.check()  # the other sequence's row is in, nothing else changed
    ctx.close()


# -------------------------------------------------------------------- together
def test_steps_on_a_side_stream_and_in_a_graph():
    """A decode loop as a program runs it: append with rotation and attend, captured once, replayed with the lengths
    moved on, on a stream of its own; each step against the plain forms of the cache as it then is."""
    rng = np.random.default_rng(32)
    dim, page, kv_heads, heads = 64, 16, 2, 4
    cache = Cache(rng, "i8", dim, page, kv_heads, [30, 5], extra_positions=8)
    table = plain_table(100, dim)
    side = torch.cuda.Stream()
    k, v = (torch.zeros(2, kv_heads, dim, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    q, q_out, out = (torch.zeros(2, heads, dim, device="cuda", dtype=torch.bfloat16) for _ in range(3))
    kv, rope = cache.on_device(), F.Rope(dev(table))
    lens = dev(np.array([30, 5], np.int32))
    batch = F.PagedBatch(dev(cache.table), lens, rows=1)
    scratch = [t.clone() for t in cache.dev]

    def step():
        lens.add_(1)
        F.paged_append(kv, batch, k, v, rope=rope, q=q, q_out=q_out)
        F.paged_attention(kv, batch, q_out, out)

    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        step()  # the stream's context is made here
    torch.cuda.synchronize()
    for t, s in zip(cache.dev, scratch):
        t.copy_(s)
    lens.copy_(dev(np.array([30, 5], np.int32)))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for i in range(6):
        x = [torch.from_numpy(rng.standard_normal(t.shape).astype(np.float32)).to(t.dtype) for t in (k, v, q)]
        for t, s in zip((k, v, q), x):
            t.copy_(s)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        cache.lens = [31 + i, 6 + i]
        at = np.array([30 + i, 5 + i])
        kx = R.rotate(x[0].double().numpy(), table, at, "interleaved", dtype=np.float32)
        R.append(cache.codes[0], cache.scales[0], kx, [1, 1], cache.lens, cache.table, "i8")
        R.append(cache.codes[1], cache.scales[1], x[1].float().numpy(), [1, 1], cache.lens, cache.table, "i8")
        cache.check()
        for b in range(2):
            o, _, size = R.attend(q_out[b].double().cpu().numpy(), cache.values(0, b), cache.values(1, b),
                                  cache.lens[b] - 1, 0, None, dim ** -0.5)
            top = np.abs(cache.values(1, b)).max()
            bound = (4 * 2.0 ** -17 * size + 2.0 ** -18 + 2.0 ** -11) * top
            assert within(out[b].double().cpu().numpy(), o, bound, "bf16")


def test_offsets_beyond_32_bits():
    """A pool of more than 2^32 bytes: the last pages are appended to and read."""
    page, kv_heads, dim = 128, 8, 128
    pages = (1 << 32) // (page * kv_heads * dim) + 40
    codes = [torch.zeros(pages, kv_heads, page, dim, dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.zeros(pages, kv_heads, device="cuda") for _ in range(2)]
    kv = F.PagedKv(*codes, *scales)
    table = dev(np.arange(pages - 1, pages - 4, -1, dtype=np.int32)[None, :])
    rng = np.random.default_rng(33)
    k, kx = rows_of(rng, 300, kv_heads, dim, "f32")
    v, vx = rows_of(rng, 300, kv_heads, dim, "f32")
    batch = F.PagedBatch(table, dev(np.array([300], np.int32)), rows=300)
    F.paged_append(kv, batch, k, v)
    q, qv = rows_of(rng, 1, kv_heads, dim, "f32")
    out = torch.empty(1, kv_heads, dim, device="cuda")
    F.paged_attention(kv, F.PagedBatch(table, dev(np.array([300], np.int32))), q, out)
    o, _, _ = R.attend(qv[0], kx.transpose(1, 0, 2), vx.transpose(1, 0, 2), 299, 0, None, dim ** -0.5)
    # Codes of 8 bits: half a step of max / 127 in every key and value.
    step = max(np.abs(kx).max(), np.abs(vx).max()) / 254
    assert np.abs(out.double().cpu().numpy()[0] - o).max() <= step * (1 + 4 * np.abs(qv).sum(-1).max() * dim ** -0.5)
    assert int(sum((c != 0).any(dim=(1, 2, 3)).sum() for c in codes)) == 6  # three pages each, nothing else


def test_example_decodes():
    """The example's loop runs, and picks the same tokens for the same seed."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_decode.py")
    spec = importlib.util.spec_from_file_location("paged_decode", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    for fmt in ("e4m3", "i8"):
        a, _ = example.decode(seqs=3, prompt=300, steps=20, fmt=fmt)
        b, _ = example.decode(seqs=3, prompt=300, steps=20, fmt=fmt)
        assert a.shape == (20, 3) and torch.equal(a, b)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_attention_query_that_is_not_finite(bad):
    """Its own row's head becomes NaN; the others are as without it."""
    rng = np.random.default_rng(34)
    for fmt, dtype in (("i8", "bf16"), ("e4m3", "f32")):
        cache = Cache(rng, fmt, 64, 16, 2, [40, 300])
        kv, batch = cache.on_device(), cache.batch([2, 2], False)
        q, _ = rows_of(rng, 4, 4, 64, dtype)
        good, out = (torch.empty_like(q) for _ in range(2))
        F.paged_attention(kv, batch, q, good)
        q[2, 1, 7] = bad
        F.paged_attention(kv, batch, q, out)
        assert out[2, 1].isnan().all()
        out[2, 1] = good[2, 1]
        assert torch.equal(out, good)


def test_attention_windows_whose_older_pages_are_gone():
    """Pages that no row of a window sees may be handed back: their table entries are not read."""
    rng = np.random.default_rng(35)
    for fmt in ("i8", "e4m3"):
        cache = Cache(rng, fmt, 64, 16, 1, [700])
        q, qv = rows_of(rng, 2, 2, 64, "f32")
        out = torch.empty_like(q)
        k, v = cache.values(0, 0), cache.values(1, 0)
        cache.table[0, :(700 - 2 - 100) // 16] = -1
        ctx = F.Context(0)
        F.paged_attention(cache.on_device(), cache.batch([2], False), q, out, window=100, ctx=ctx)
        ctx.synchronize()
        for r in range(2):
            o, _, size = R.attend(qv[r], k, v, 698 + r, 100, None, 0.125)
            top = np.abs(v).max()
            assert within(out[r].double().cpu().numpy(), o, (4 * 2.0 ** -17 * size + 2.0 ** -18) * top, "f32")
        ctx.close()


def test_attention_more_sequences_than_a_block_has_threads():
    """The schedule in pieces: 1,100 sequences of up to a few pages, some without a position."""
    lens = [int(n) for n in np.random.default_rng(1).integers(0, 40, 1100)]
    attention_case(36, "i8", 64, 16, 1, 2, "bf16", lens, [1] * 1100)
    attention_case(37, "e4m3", 64, 16, 2, 1, "f32", lens[:33], [1] * 33)


def test_positions_near_two_to_the_31():
    """A table with room for nearly 2^31 positions (one sequence whose older pages are gone): rows are appended to its
    last pages and a window over the last tile is read, without an index that wraps."""
    page, room = 16, (2 ** 31 - 1) // 16
    last, rows, kv_heads, dim = room * page, 32, 2, 64
    table = torch.full((1, room), -1, dtype=torch.int32, device="cuda")
    table[0, -6:] = torch.arange(6, dtype=torch.int32, device="cuda")
    for fmt, kind in (("i8", torch.int8), ("e4m3", torch.float8_e4m3fn)):
        rng = np.random.default_rng(50)
        # One page more than the table names, which stays as it is.
        codes = [np.zeros((7, kv_heads, page, dim), np.uint8) for _ in range(2)]
        scales = [np.zeros((7, kv_heads), np.float32) for _ in range(2)]
        on_device = [dev(c).view(kind) for c in codes] + [dev(s) for s in scales]
        kv = F.PagedKv(*on_device)
        x = [rows_of(rng, 6 * page, kv_heads, dim, "f32") for _ in range(2)]
        ctx = F.Context(0)
        for to in (last - 2 * rows, last - rows, last):
            at = 6 * page - (last - to) - rows
            part = slice(at, at + rows)
            F.paged_append(kv, F.PagedBatch(table, dev(np.array([to], np.int32)), rows=rows,
                                            row_start=dev(np.array([0, rows], np.int32))), x[0][0][part], x[1][0][part],
                           ctx=ctx)
            for i in range(2):
                R.append(codes[i], scales[i], x[i][1][part].astype(np.float32), [rows], [at + rows], np.arange(6)[None],
                         fmt)
        ctx.synchronize()
        for i in range(2):
            assert np.array_equal(on_device[i].view(torch.uint8).cpu().numpy(), codes[i])
            assert np.array_equal(on_device[2 + i].cpu().numpy(), scales[i])
        k, v = ((R.decode(c[:6], fmt) * s[:6, :, None, None].astype(np.float64)).transpose(1, 0, 2, 3).reshape(
            kv_heads, -1, dim) for c, s in zip(codes, scales))
        for n in (1, 3):
            q, qv = rows_of(rng, n, 4, dim, "f32")
            out = torch.empty_like(q)
            F.paged_attention(kv, F.PagedBatch(table, dev(np.array([last], np.int32)), rows=n), q, out, window=50,
                              ctx=ctx)
            ctx.synchronize()
            for r in range(n):
                o, _, size = R.attend(qv[r], k, v, 6 * page - n + r, 50, None, dim ** -0.5)
                bound = (4 * 2.0 ** -17 * size + 2.0 ** -18) * np.abs(v).max()
                assert within(out[r].double().cpu().numpy(), o, bound, "f32")
        ctx.close()


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("number", [-1, -7, -(1 << 31), "pages", 1 << 30])
def test_attention_reports_every_page_number_outside_the_pool(fmt, number):
    """-1, the usual mark of a place that has no page, among them: where rows see it the error word says so and they
    are NaN; the other sequences are whole."""
    rng = np.random.default_rng(40)
    for dim, lens, bad in ((64, [40, 200, 9], 3), (128, [500, 333], 0)):
        cache = Cache(rng, fmt, dim, 16, 2, lens)
        q, qv = rows_of(rng, len(lens), 4, dim, "bf16")
        out, lse = torch.full_like(q, 9.0), torch.full((len(lens), 4), 9.0, device="cuda")
        cache.table[1, bad] = cache.codes[0].shape[0] if number == "pages" else number
        ctx = F.Context(0)
        F.paged_attention(cache.on_device(), cache.batch([1] * len(lens), False), q, out, lse=lse, ctx=ctx)
        with pytest.raises(F.FoError, match="page table"):
            ctx.synchronize()
        ctx.synchronize()  # reported once
        assert out[1].isnan().all() and lse[1].isnan().all()
        for b in range(len(lens)):
            if b == 1:
                continue
            o, _, size = R.attend(qv[b], cache.values(0, b), cache.values(1, b), lens[b] - 1, 0, None, dim ** -0.5)
            top = np.abs(cache.values(1, b)).max()
            bound = (4 * 2.0 ** -17 * size + 2.0 ** -18 + 2.0 ** -11) * top
            assert within(out[b].double().cpu().numpy(), o, bound, "bf16")
        ctx.close()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_rows_that_see_nothing_whatever_they_hold(bad, fmt, dtype):
    """A padded slot's queries are whatever its buffer was left with: 0 and -infinity all the same, and nothing of
    them reaches the other rows."""
    rng = np.random.default_rng(41)
    for dim, group, rows, lens, window in ((64, 2, 1, [0, 300, 0], 0), (128, 1, 5, [3, 0, 700], 0),
                                           (64, 5, 5, [2, 0, 90], 16), (128, 8, 7, [2500, 6], 0)):
        cache = Cache(rng, fmt, dim, 16, 2, lens)
        kv, batch = cache.on_device(), cache.batch([rows] * len(lens), False)
        q, _ = rows_of(rng, rows * len(lens), 2 * group, dim, dtype)
        sinks = dev(rng.standard_normal(2 * group).astype(np.float32))
        empty = [b * rows + r for b, n in enumerate(lens) for r in range(rows) if n - rows + r < 0]
        good, out = (torch.full_like(q, 9.0) for _ in range(2))
        lses = [torch.full((q.shape[0], 2 * group), 9.0, device="cuda") for _ in range(2)]
        F.paged_attention(kv, batch, q, good, sinks=sinks, window=window, lse=lses[0])
        q[empty] = bad
        F.paged_attention(kv, batch, q, out, sinks=sinks, window=window, lse=lses[1])
        assert torch.equal(out, good) and torch.equal(lses[1], lses[0])
        assert (out[empty] == 0).all() and (lses[1][empty] == -math.inf).all()


def test_padded_slots_from_append_to_attention():
    """A captured graph's padded slot (length 0) with NaN left in its rows, through a whole step."""
    rng = np.random.default_rng(42)
    for fmt in ("i8", "e4m3"):
        cache = Cache(rng, fmt, 64, 16, 2, [0, 20], extra_positions=1)
        kv = cache.on_device()
        cache.lens = [0, 21]
        batch = cache.batch([1, 1], False)
        k, v = (rows_of(rng, 2, 2, 64, "bf16")[0] for _ in range(2))
        q, _ = rows_of(rng, 2, 4, 64, "bf16")
        for t in (k, v, q):
            t[0] = math.nan
        q_out, out = (torch.full_like(q, 9.0) for _ in range(2))
        ctx = F.Context(0)
        F.paged_append(kv, batch, k, v, rope=F.Rope(dev(plain_table(40, 64))), q=q, q_out=q_out, ctx=ctx)
        F.paged_attention(kv, batch, q_out, out, ctx=ctx)
        ctx.synchronize()
        assert (out[0] == 0).all() and out[1].isfinite().all() and (out[1] != 0).any()
        ctx.close()


def test_reports_touch_their_own_stream_alone():
    """A report reads and clears the error word, and after a bounded wait the attention's counters, in the order of the
    context's stream: work on the default stream neither delays it nor can be overtaken by it."""
    side = torch.cuda.Stream()
    rng = np.random.default_rng(43)
    cache = Cache(rng, "i8", 64, 16, 1, [9000])
    q, _ = rows_of(rng, 1, 1, 64, "f32")
    outs = [torch.empty_like(q) for _ in range(2)]
    kv, batch = cache.on_device(), cache.batch([1], False)
    ctx = F.Context(0, side.cuda_stream)
    torch.cuda.synchronize()
    F.paged_attention(kv, batch, q, outs[0], ctx=ctx)
    assert ctx.selftest_bounded_wait(1000) == F.ERR_CUDA
    torch.cuda.synchronize()
    torch.cuda._sleep(int(1e9))  # half a second on the default stream
    busy = torch.cuda.Event()
    busy.record()
    assert ctx.selftest_bounded_wait(1000) == F.ERR_CUDA
    F.paged_attention(kv, batch, q, outs[1], ctx=ctx)
    ctx.synchronize()
    assert not busy.query()
    assert torch.equal(*outs)
    torch.cuda.synchronize()
    ctx.close()


def test_a_batch_plan_tells_other_calls_errors_apart():
    """A paged call's error that is still unread when a plan on the same context finishes is reported as what it is."""
    import generators as G
    ctx = F.Context(0)
    k, v, _ = G.kv_fixture(300, 21)
    cache = F.SplitPrefix.from_compact(dev(k), dev(v), 300, 308, fmt=F.KV_Q8, ctx=ctx)
    rows = [[torch.zeros(1024, device="cuda")] for _ in range(4)]
    plan = F.BatchPlan([cache], *rows[:3], [torch.zeros(16, device="cuda")], rows[3])
    plan.step()
    x = torch.ones(1, 2, 64, device="cuda")
    F.rope(x, torch.empty_like(x), F.Rope(dev(plain_table(4, 64))), dev(np.array([4], np.int32)), ctx=ctx)
    with pytest.raises(F.FoError, match="outside its table"):
        plan.finish()
    ctx.synchronize()  # reported once
    assert cache.tail_len == 1
    cache.close()
    ctx.close()


@pytest.mark.parametrize("per", [2, 30])
def test_rows_of_no_sequence(per):
    """Rows before the first sequence's and behind the last one's: their queries are copied as they are, nothing of
    them is stored or reported, and the attention leaves their outputs alone."""
    rng = np.random.default_rng(44)
    start = [3, 3 + per, 3 + per, 3 + 2 * per]
    total, held, rows = start[-1] + 40, [10, 5, 0], [per, 0, per]
    cache = Cache(rng, "i8", 64, 16, 2, held, extra_positions=per)
    kv = cache.on_device()
    cache.lens = [n + m for n, m in zip(held, rows)]
    batch = F.PagedBatch(dev(cache.table), dev(np.array(cache.lens, np.int32)), rows=per,
                         row_start=dev(np.array(start, np.int32)))
    table = plain_table(10 + per, 64)  # no position beyond the longest sequence's
    k, kx = rows_of(rng, total, 2, 64, "f32")
    v, vx = rows_of(rng, total, 2, 64, "f32")
    q, qx = rows_of(rng, total, 4, 64, "f32")
    q_out, out = (torch.full_like(q, 5.0) for _ in range(2))
    lse = torch.full((total, 4), 5.0, device="cuda")
    own = np.array(list(range(start[0], start[1])) + list(range(start[2], start[3])))
    others = np.setdiff1d(np.arange(total), own)
    k[others], v[others] = math.nan, math.inf
    ctx = F.Context(0)
    F.paged_append(kv, batch, k, v, rope=F.Rope(dev(table)), q=q, q_out=q_out, ctx=ctx)
    F.paged_attention(kv, batch, q_out, out, lse=lse, ctx=ctx)
    ctx.synchronize()
    at = np.concatenate([np.arange(n, n + m) for n, m in zip(held, rows)])
    kr = R.rotate(kx[own], table, at, "interleaved", dtype=np.float32)
    R.append(cache.codes[0], cache.scales[0], kr.astype(np.float32), rows, cache.lens, cache.table, "i8")
    R.append(cache.codes[1], cache.scales[1], vx[own].astype(np.float32), rows, cache.lens, cache.table, "i8")
    cache.check()
    expected = qx.astype(np.float32)
    expected[own] = R.rotate(qx[own], table, at, "interleaved", dtype=np.float32)
    assert np.array_equal(q_out.cpu().numpy(), expected)
    assert (out[others] == 5).all() and (lse[others] == 5).all()
    assert (out[own] != 5).all() and lse[own].isfinite().all()
    # Positions that are given hold for every row.
    where = dev((np.arange(total) % (10 + per)).astype(np.int32))
    F.paged_append(kv, batch, k, v, rope=F.Rope(dev(table)), positions=where, q=q, q_out=q_out, ctx=ctx)
    ctx.synchronize()
    expected = R.rotate(qx, table, np.arange(total) % (10 + per), "interleaved", dtype=np.float32)
    assert np.array_equal(q_out.cpu().numpy(), expected)
    ctx.close()


def test_first_use_while_a_graph_is_captured(monkeypatch):
    """A stream's context and its attention's scratch cannot be made inside a capture: the call says so, before it
    launches or allocates anything, and works once they are there."""
    rng = np.random.default_rng(45)
    cache = Cache(rng, "i8", 64, 16, 1, [40])
    kv, batch = cache.on_device(), cache.batch([1], False)
    q, _ = rows_of(rng, 1, 2, 64, "f32")
    expected, out = torch.empty_like(q), torch.zeros_like(q)
    F.paged_attention(kv, batch, q, expected)
    monkeypatch.setattr(F, "_stream_contexts", {})
    side = torch.cuda.Stream()
    torch.cuda.synchronize()

    def refused():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            with pytest.raises(F.FoError, match="captur"):
                F.paged_attention(kv, batch, q, out)
            out.add_(0.0)  # the capture itself goes on
        graph.replay()
        torch.cuda.synchronize()

    refused()  # no context
    with torch.cuda.stream(side):
        F.rope(q, torch.empty_like(q), F.Rope(dev(plain_table(4, 64))))
    refused()  # a context that no attention has run on
    with torch.cuda.stream(side):
        F.paged_attention(kv, batch, q, out)
    torch.cuda.synchronize()
    out.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        F.paged_attention(kv, batch, q, out)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, expected)


def test_first_attentions_of_a_context_from_several_threads():
    """They make its scratch once."""
    import threading
    rng = np.random.default_rng(46)
    cache = Cache(rng, "i8", 64, 16, 2, [5000, 40])
    kv = cache.on_device()
    batches = [cache.batch([1, 1], False) for _ in range(8)]
    q, _ = rows_of(rng, 2, 4, 64, "f32")
    expected = torch.empty_like(q)
    F.paged_attention(kv, cache.batch([1, 1], False), q, expected)
    torch.cuda.synchronize()
    for _ in range(5):
        ctx = F.Context(0)
        outs = [torch.zeros_like(q) for _ in batches]
        gate = threading.Barrier(len(batches))
        failures = []

        def call(batch, out):
            gate.wait()
            try:
                F.paged_attention(kv, batch, q, out, ctx=ctx)
            except Exception as e:  # noqa: BLE001
                failures.append(e)

        threads = [threading.Thread(target=call, args=a) for a in zip(batches, outs)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        ctx.synchronize()
        assert not failures
        assert all(torch.equal(o, expected) for o in outs)
        ctx.close()


def test_calls_without_rows():
    """Empty batches (torch gives their tensors no memory) do nothing."""
    kv = F.PagedKv(*(torch.ones(3, 2, 16, 64, dtype=torch.int8, device="cuda") for _ in range(2)),
                   *(torch.ones(3, 2, device="cuda") for _ in range(2)))
    rope = F.Rope(dev(plain_table(4, 64)))
    ints = dict(dtype=torch.int32, device="cuda")
    ctx = F.Context(0)
    for batch in (F.PagedBatch(torch.zeros(0, 2, **ints), torch.zeros(0, **ints)),
                  F.PagedBatch(torch.zeros(0, 2, **ints), torch.zeros(0, **ints), row_start=torch.zeros(1, **ints)),
                  F.PagedBatch(torch.zeros(2, 2, **ints), torch.zeros(2, **ints), row_start=torch.zeros(3, **ints)),
                  F.PagedBatch(torch.zeros(2, 2, **ints), torch.zeros(2, **ints), rows=0)):
        for dtype in DTYPES.values():
            q, k = torch.empty(0, 4, 64, dtype=dtype, device="cuda"), torch.empty(0, 2, 64, dtype=dtype, device="cuda")
            F.rope(q, q, rope, ctx=ctx)
            F.paged_append(kv, batch, k, k, rope=rope, q=q, q_out=torch.empty_like(q), ctx=ctx)
            F.paged_attention(kv, batch, q, torch.empty_like(q), lse=torch.empty(0, 4, device="cuda"), ctx=ctx)
    ctx.synchronize()
    assert all((t.float() == 1).all() for t in kv.keep)
    ctx.close()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_queries_with_one_large_element(dim, dtype):
    """One element 2^7 times the others, in a dimension where all keys are 0: the scores come from the others, and are
    as exact as without it (the bound on a score, 2^-17 of its sum of magnitudes).  FP32 rows hold an element to 2^-22 of
    their largest one, which adds that to each product."""
    rng = np.random.default_rng(47)
    for n in (8, 500):
        cache = Cache(rng, "i8", dim, 16, 2, [n])
        cache.codes[0][..., 5] = 0
        kv, batch = cache.on_device(), cache.batch([1], False)
        q, _ = rows_of(rng, 1, 6, dim, dtype)
        q[..., 5] = 128.0 * q.abs().amax(-1)
        qv = q.double().cpu().numpy()
        out, lse = torch.empty_like(q), torch.empty(1, 6, device="cuda")
        F.paged_attention(kv, batch, q, out, lse=lse)
        k, v = cache.values(0, 0), cache.values(1, 0)
        o, z, size = R.attend(qv[0], k, v, n - 1, 0, None, dim ** -0.5)
        d, top = 2.0 ** -17 * size, np.abs(v).max()
        if dtype == "f32":
            d += 2.0 ** -22 * np.abs(qv).max() * np.abs(k).sum(-1).max() * dim ** -0.5
        assert (np.abs(lse[0].double().cpu().numpy() - z) <= d + 2.0 ** -20 * (1 + np.abs(z))).all()
        bound = (4 * d + 2.0 ** -18 + (2.0 ** -11 if dtype == "bf16" else 0)) * top
        assert within(out[0].double().cpu().numpy(), o, bound, dtype)


@pytest.mark.parametrize("nats", [2.0, 5.0, 8.0, 12.0, 15.0])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_attention_large_weights_with_small_values(nats, dtype, fmt):
    """Keys that take nearly all of the softmax and whose values are zero (as a text's first tokens often do): what is
    left of the output is the other keys', and their probabilities have to be exact to their own size.  Each
    probability keeps 8 bits with BF16 rows (a relative 2^-9 and, where all keys of a group are like one another, at
    most twice that) and 15 with FP32 rows; a score is off by d at most, which moves a probability and the sum by e^d
    each; FP32 sums add 2^-18."""
    rng = np.random.default_rng(48)
    kept = 2.0 ** (-8 if dtype == "bf16" else -15 if fmt == "i8" else -13)
    for dim, n, large in ((64, 2, 1), (128, 3, 1), (64, 7, 2), (64, 60, 1), (64, 64, 4), (64, 2000, 1), (128, 30, 1),
                          (128, 777, 4)):
        cache = Cache(rng, fmt, dim, 64, 1, [n])
        pages = cache.table[0, :-(-n // 64)]
        sign = np.where(rng.standard_normal(dim) < 0, -1.0, 1.0)
        q = torch.from_numpy((sign * rng.uniform(0.5, 1.5, (1, 2, dim))).astype(np.float32)).to(DTYPES[dtype]).cuda()
        qv = q.double().cpu().numpy()
        # Keys near zero, but for the first ones, whose scores are `nats` above with the first query.
        unit = nats / (127.0 * dim ** -0.5 * np.abs(qv[0, 0]).sum())
        small = R.encode(rng.integers(-12, 13, cache.codes[0].shape).astype(np.float32), fmt)
        cache.codes[0][:] = small
        cache.codes[0][pages[0], :, :large] = R.encode((127.0 if fmt == "i8" else 128.0) * sign.astype(np.float32), fmt)
        cache.codes[1][pages[0], :, :large] = 0
        cache.scales[0][pages] = np.float32(unit)
        out, lse = torch.empty_like(q), torch.empty(1, 2, device="cuda")
        F.paged_attention(cache.on_device(), cache.batch([1], False), q, out, lse=lse)
        k, v = cache.values(0, 0), cache.values(1, 0)
        o, z, size = R.attend(qv[0], k, v, n - 1, 0, None, dim ** -0.5)
        sizes, _, _ = R.attend(qv[0], k, np.abs(v), n - 1, 0, None, dim ** -0.5)
        d = 2.0 ** -17 * size
        bound = (2 * (math.exp(d) - 1) + kept + 2.0 ** -18) * sizes
        assert within(out[0].double().cpu().numpy(), o, bound, dtype)
        assert (np.abs(lse[0].double().cpu().numpy() - z) <= d + 2.0 ** -20 * (1 + np.abs(z))).all()


def test_attention_from_a_thread_without_cuda_calls_before_it():
    """A server's worker thread, whose first CUDA call of any kind is an attention on a context that others made."""
    import threading
    rng = np.random.default_rng(51)
    cache = Cache(rng, "e4m3", 64, 16, 2, [300])
    kv, batch = cache.on_device(), cache.batch([1], False)
    q, _ = rows_of(rng, 1, 4, 64, "bf16")
    expected, out = (torch.zeros_like(q) for _ in range(2))
    ctx = F.Context(0)
    F.paged_attention(kv, batch, q, expected, ctx=ctx)
    failures = []

    def call():
        try:
            F.paged_attention(kv, batch, q, out, ctx=ctx)
        except Exception as e:  # noqa: BLE001
            failures.append(e)

    worker = threading.Thread(target=call)
    worker.start()
    worker.join()
    ctx.synchronize()
    assert not failures and torch.equal(out, expected)
    ctx.close()


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_offsets_beyond_32_bits_bit_for_bit(fmt):
    """A pool of more than 2^32 bytes: rows appended to its last pages are there, code for code, nothing is anywhere
    else, and the attention over them is as exact as over any."""
    page, kv_heads, dim, held = 128, 8, 128, 300
    pages = (1 << 32) // (page * kv_heads * dim) + 40
    kind = torch.int8 if fmt == "i8" else torch.float8_e4m3fn
    codes = [torch.zeros(pages, kv_heads, page, dim, dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.zeros(pages, kv_heads, device="cuda") for _ in range(2)]
    kv = F.PagedKv(*(c.view(kind) for c in codes), *scales)
    ids = np.arange(pages - 1, pages - 4, -1, dtype=np.int32)
    rng = np.random.default_rng(49)
    k, kx = rows_of(rng, held, kv_heads, dim, "f32")
    v, vx = rows_of(rng, held, kv_heads, dim, "f32")
    F.paged_append(kv, F.PagedBatch(dev(ids[None]), dev(np.array([held], np.int32)), rows=held), k, v)
    F.paged_append(kv, F.PagedBatch(dev(ids[None]), dev(np.array([held + 1], np.int32))), k[:1], v[:1])  # one row more
    values = []
    for i, x in enumerate((kx, vx)):
        c, s = np.zeros((3, kv_heads, page, dim), np.uint8), np.zeros((3, kv_heads), np.float32)
        R.append(c, s, x.astype(np.float32), [held], [held], np.array([[0, 1, 2]]), fmt)
        R.append(c, s, x[:1].astype(np.float32), [1], [held + 1], np.array([[0, 1, 2]]), fmt)
        assert np.array_equal(codes[i][ids.astype(np.int64)].view(torch.uint8).cpu().numpy(), c)
        assert np.array_equal(scales[i][ids.astype(np.int64)].cpu().numpy(), s)
        assert not codes[i][:pages - 3].any() and not scales[i][:pages - 3].any()
        values.append((R.decode(c, fmt) * s[..., None, None].astype(np.float64)).transpose(1, 0, 2, 3).reshape(
            kv_heads, -1, dim)[:, :held + 1])
    q, qv = rows_of(rng, 1, kv_heads, dim, "f32")
    out = torch.empty(1, kv_heads, dim, device="cuda")
    F.paged_attention(kv, F.PagedBatch(dev(ids[None]), dev(np.array([held + 1], np.int32))), q, out)
    o, _, size = R.attend(qv[0], *values, held, 0, None, dim ** -0.5)
    bound = (4 * 2.0 ** -17 * size + 2.0 ** -18) * np.abs(values[1]).max()
    assert within(out[0].double().cpu().numpy(), o, bound, "f32")
