"""Refusals of the rotary and paged-cache entry points, on the host before
any device call, and the plain implementations that the GPU tests use."""

import ctypes

import numpy as np
import pytest

import fo_cuda as F
import paged_reference as R


def last_error():
    return F.lib().fo_last_error().decode()


BUF = np.zeros(1 << 16, np.float32)
BASE = (BUF.ctypes.data + 255) & ~255


def rows(heads=8, dtype=0, row_stride=512, head_stride=64, data=BASE):
    return F.Rows(data, row_stride, head_stride, heads, dtype)


def pool(**change):
    p = dict(k_codes=BASE, v_codes=BASE, k_scales=BASE, v_scales=BASE, n_pages=4, page_size=16, n_kv_heads=8,
             head_dim=64, format=0)
    p.update(change)
    return F.PagedPool(*p.values())


def batch(**change):
    b = dict(page_table=BASE, lens=BASE, row_start=None, table_stride=2, n_seqs=2, max_rows=1, total_rows=2)
    b.update(change)
    return F.PagedSequences(*b.values())


def spec(**change):
    s = dict(table=BASE, positions=16, row_positions=None, rot_dim=64, layout=0)
    s.update(change)
    return F.RopeSpec(*s.values())


def ref(x):
    return None if x is None else ctypes.byref(x)


def rope(x=rows(), out=rows(), n=2, dim=64, s=spec(), transpose=0):
    return F.lib().fo_rope(None, ref(x), ref(out), n, dim, ref(s), transpose)


def append(kv=pool(), b=batch(), k=rows(), v=rows(), q=None, q_out=None, s=None):
    return F.lib().fo_paged_append(None, ref(kv), ref(b), ref(k), ref(v), ref(q), ref(q_out), ref(s))


def attend(kv=pool(), b=batch(), q=rows(16, row_stride=1024), out=rows(16, row_stride=1024), sinks=None, scale=0.125,
           window=0, lse=None):
    return F.lib().fo_paged_attention(None, ref(kv), ref(b), ref(q), sinks, scale, window, ref(out), lse)


@pytest.mark.parametrize("call,message", [
    (lambda: rope(x=None), "null pointer"),
    (lambda: rope(x=rows(data=None)), "null pointer"),
    (lambda: rope(x=rows(dtype=2)), "unknown type"),
    (lambda: rope(x=rows(heads=0)), "head count"),
    (lambda: rope(x=rows(row_stride=-1)), "negative stride"),
    (lambda: rope(x=rows(data=BASE + 2)), "misaligned"),
    (lambda: rope(x=rows(dtype=1, data=BASE + 1)), "misaligned"),
    (lambda: rope(out=rows(row_stride=0)), "rows overlap"),
    (lambda: rope(out=rows(row_stride=64, head_stride=64)), "rows overlap"),
    (lambda: rope(out=rows(head_stride=32)), "rows overlap"),
    (lambda: rope(x=rows(heads=7)), "as many heads"),
    (lambda: rope(x=rows(dtype=1)), "one type"),
    (lambda: rope(x=rows(row_stride=1024)), "laid out alike"),
    (lambda: rope(n=-1), "rows must be"),
    (lambda: rope(dim=257), "head_dim"),
    (lambda: rope(s=None), "null table"),
    (lambda: rope(s=spec(table=BASE + 4)), "8-byte aligned"),
    (lambda: rope(s=spec(positions=0)), "without positions"),
    (lambda: rope(s=spec(rot_dim=66)), "rot_dim"),
    (lambda: rope(s=spec(rot_dim=3)), "rot_dim"),
    (lambda: rope(s=spec(layout=2)), "unknown layout"),
    (lambda: rope(), "null context"),
    (lambda: append(kv=None), "null descriptor"),
    (lambda: append(b=None), "null descriptor"),
    (lambda: append(kv=pool(page_size=48)), "page_size"),
    (lambda: append(kv=pool(head_dim=96)), "head_dim must be"),
    (lambda: append(kv=pool(format=2)), "unknown format"),
    (lambda: append(kv=pool(n_kv_heads=0)), "KV heads"),
    (lambda: append(kv=pool(n_pages=0)), "pages must be"),
    (lambda: append(kv=pool(v_scales=None)), "null pool"),
    (lambda: append(kv=pool(k_codes=BASE + 8)), "16-byte aligned"),
    (lambda: append(b=batch(n_seqs=-1)), "at most 65,535"),
    (lambda: append(b=batch(total_rows=3)), "total_rows must be"),
    (lambda: append(b=batch(lens=None)), "null page table"),
    (lambda: append(b=batch(table_stride=0)), "1 page to"),
    (lambda: append(b=batch(lens=BASE + 2)), "misaligned integers"),
    (lambda: append(k=rows(heads=4)), "cache's heads"),
    (lambda: append(v=rows(dtype=1)), "one type"),
    (lambda: append(q=rows(), s=spec()), "q needs q_out"),
    (lambda: append(q=rows(), q_out=rows()), "without rope"),
    (lambda: append(q=rows(), q_out=rows(dtype=1), s=spec()), "one type"),
    (lambda: append(s=spec(rot_dim=128)), "rot_dim"),
    (lambda: append(), "null context"),
    (lambda: attend(q=rows(12, row_stride=1024)), "as many heads"),
    (lambda: attend(q=rows(12, row_stride=1024), out=rows(12, row_stride=1024)), "multiple of the KV heads"),
    (lambda: attend(b=batch(max_rows=65, total_rows=130)), "at most 64 rows"),
    (lambda: attend(scale=float("inf")), "finite"),
    (lambda: attend(window=-1), "negative window"),
    (lambda: attend(lse=BASE + 2), "misaligned"),
    (lambda: attend(out=rows(16, row_stride=512)), "rows overlap"),
    (lambda: attend(), "null context"),
])
def test_refusals(call, message):
    assert call() == F.ERR_INVALID
    assert message in last_error()


def test_tables_with_room_for_too_many_tiles():
    many = batch(n_seqs=60000, total_rows=60000, table_stride=(1 << 31) // 128 - 1)
    assert attend(b=many) == F.ERR_CAPACITY and "2^31 tiles" in last_error()


@pytest.mark.parametrize("change", [
    dict(theta=1.0), dict(theta=float("nan")), dict(scaling=4), dict(scaling=1, factor=0.0),
    dict(scaling=3, original_positions=0.0), dict(scaling=3, beta_slow=0.0), dict(scaling=3, beta_fast=0.5),
    dict(scaling=3, attention_factor=-1.0),
])
def test_table_refusals(change):
    s = dict(theta=10000.0, scaling=0, factor=2.0, original_positions=4096.0, beta_fast=32.0, beta_slow=1.0,
             attention_factor=0.0)
    s.update(change)
    assert F.lib().fo_rope_table(None, BASE, 16, 64, F.RopeScaling(*s.values())) == F.ERR_INVALID
    assert "fo_rope_table" in last_error()
    good = F.RopeScaling(10000.0, 3, 2.0, 4096.0, 32.0, 1.0, 0.0)
    for table, n, rot in ((None, 16, 64), (BASE + 4, 16, 64), (BASE, 0, 64), (BASE, 16, 63), (BASE, 16, 258)):
        assert F.lib().fo_rope_table(None, table, n, rot, good) == F.ERR_INVALID
    assert F.lib().fo_rope_table(None, BASE, 16, 64, good) == F.ERR_INVALID and last_error() == "null context"


def test_bindings_refuse_what_is_not_on_the_device():
    torch = pytest.importorskip("torch")
    t = torch.zeros(2, 8, 64)
    with pytest.raises(F.FoError, match="CUDA tensor"):
        F.rope(t, t, None)
    with pytest.raises(F.FoError, match="rope table"):
        F.Rope(torch.zeros(4, 32, 2))
    codes = torch.zeros(4, 8, 16, 64, dtype=torch.int8)
    with pytest.raises(F.FoError, match="CUDA"):
        F.PagedKv(codes, codes, torch.zeros(4, 8), torch.zeros(4, 8))
    with pytest.raises(F.FoError, match="int8 or float8"):
        F.PagedKv(codes.float(), codes.float(), torch.zeros(4, 8), torch.zeros(4, 8))
    with pytest.raises(F.FoError, match="keys and values alike"):
        F.PagedKv(codes, codes[:2], torch.zeros(4, 8), torch.zeros(4, 8))
    with pytest.raises(F.FoError, match="one length"):
        F.PagedBatch(torch.zeros(2, 4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32))


def test_plain_codes():
    """The plain e4m3 rounding against torch's, every code and the ties between neighbours."""
    torch = pytest.importorskip("torch")
    v = R.E4M3[:127]
    x = np.concatenate((v, (v[1:] + v[:-1]) / 2, np.random.default_rng(0).uniform(0, 448, 5000)))
    x = np.concatenate((x, -x)).astype(np.float32)
    theirs = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(R.encode(x, "e4m3"), theirs)
    assert np.array_equal(R.encode(np.array([0.5, 1.5, -2.5, 126.6], np.float32), "i8").view(np.int8), [0, 2, -2, 127])


def test_plain_append_against_the_definition():
    """A page's codes stand for the appended values within half a step of its last scale per re-rounding."""
    rng = np.random.default_rng(1)
    codes, scales = np.zeros((3, 1, 16, 64), np.uint8), np.zeros((3, 1), np.float32)
    x = rng.standard_normal((40, 1, 64)).astype(np.float32) * np.linspace(0.2, 3, 40, dtype=np.float32)[:, None, None]
    table = np.array([[2, 0, 1]])
    for n in range(1, 41):
        R.append(codes, scales, x[n - 1:n], [1], [n], table, "i8")
    for p in range(40):
        pg = table[0, p // 16]
        got = R.decode(codes[pg, 0, p % 16], "i8") * scales[pg, 0]
        assert np.abs(got - x[p, 0]).max() <= scales[pg, 0] * 0.5 * 16
    whole, ws = np.zeros_like(codes), np.zeros_like(scales)
    R.append(whole, ws, x, [40], [40], table, "i8")
    assert np.array_equal(ws, scales)


@pytest.mark.parametrize("change", [
    dict(n_seqs=0, row_start=BASE, total_rows=5, max_rows=5), dict(n_seqs=0, row_start=BASE, total_rows=200, max_rows=64),
    dict(n_seqs=0, row_start=BASE, total_rows=5, max_rows=5, page_table=None, lens=None),
    dict(n_seqs=2, row_start=BASE, total_rows=5, max_rows=0),
])
def test_rows_without_sequences_are_refused(change):
    """Rows that no sequence could have (the kernels would look for lengths that are not there, or launch no block)."""
    b = batch(**change)
    for status in (append(b=b), append(b=b, q=rows(), q_out=rows(), s=spec()), attend(b=b)):
        assert status == F.ERR_INVALID and "rows without a sequence" in last_error()


def test_overlapped_kernels_make_no_read_only_loads():
    """A kernel that starts while the one before it ends may not load through the read-only path: it asks for memory
    that nothing writes while the kernel lives, and its life begins before the other's stores."""
    import os
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "falcon-ocr-cpu_b200", "csrc")
    files = {name: open(os.path.join(csrc, name)).read() for name in sorted(os.listdir(csrc))
             if name.endswith((".cu", ".cuh"))}
    overlapped = {name for name, text in files.items() if "wait_for_prior_kernel" in text}
    grown = True
    while grown:  # and what they include
        more = {name for name in files for user in overlapped if '#include "%s"' % name in files[user]}
        grown = not more <= overlapped
        overlapped |= more
    assert {"paged.cuh", "paged_rope.cuh", "rope.cu", "paged_append.cu", "paged_attention.cu"} <= overlapped
    for name in overlapped:
        for word in ("__ldg(", "ld.global.nc", "__restrict__"):
            assert word not in files[name], (name, word)


class DeviceTensor:
    """What the bindings ask of a CUDA tensor, on whichever GPU."""
    is_cuda = True
    __module__ = "torch"  # by which the bindings tell torch's tensors

    def __init__(self, shape, dtype, device=0):
        self.shape, self.dtype, self.index = tuple(shape), dtype, device
        self.device = self
        self.__cuda_array_interface__ = {}

    def dim(self):
        return len(self.shape)

    def numel(self):
        return int(np.prod(self.shape))

    def size(self, i):
        return self.shape[i]

    def stride(self, i=None):
        s = tuple(int(np.prod(self.shape[j + 1:])) for j in range(len(self.shape)))
        return s if i is None else s[i]

    def get_device(self):
        return self.index

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return BASE


class NoContext:
    handle, device = None, 0


def device_call(call, **other):
    """One of the paged calls, all its tensors on GPU 0 but those named."""
    torch = pytest.importorskip("torch")

    def t(name, shape, dtype=torch.float32):
        return DeviceTensor(shape, dtype, other.get(name, 0))

    ints = torch.int32
    rope = F.Rope(t("table", (16, 32, 2)))
    kv = F.PagedKv(t("k_codes", (4, 8, 16, 64), torch.int8), t("v_codes", (4, 8, 16, 64), torch.int8),
                   t("k_scales", (4, 8)), t("v_scales", (4, 8)))
    batch = F.PagedBatch(t("page_table", (2, 2), ints), t("lens", (2,), ints), row_start=t("row_start", (3,), ints))
    if call == "rope":
        F.rope(t("q", (2, 16, 64)), t("out", (2, 16, 64)), rope, t("positions", (2,), ints), ctx=NoContext)
    elif call == "append":
        F.paged_append(kv, batch, t("k", (2, 8, 64)), t("v", (2, 8, 64)), rope, t("positions", (2,), ints),
                       t("q", (2, 16, 64)), t("q_out", (2, 16, 64)), ctx=NoContext)
    else:
        F.paged_attention(kv, batch, t("q", (2, 16, 64)), t("out", (2, 16, 64)), t("sinks", (16,)), lse=t("lse", (2, 16)),
                          ctx=NoContext)


@pytest.mark.parametrize("call,names", [
    ("rope", ["table", "out", "positions"]),
    ("append", ["k_codes", "v_codes", "k_scales", "v_scales", "page_table", "lens", "row_start", "k", "v", "table",
                "positions", "q", "q_out"]),
    ("attend", ["k_codes", "v_codes", "k_scales", "v_scales", "page_table", "lens", "row_start", "q", "out", "sinks",
                "lse"]),
])
def test_bindings_refuse_tensors_of_another_gpu(call, names):
    with pytest.raises(F.FoError, match="null context"):  # all on one: taken
        device_call(call)
    for name in names:
        with pytest.raises(F.FoError, match="GPU"):
            device_call(call, **{name: 1})


def test_append_refuses_positions_without_a_rotation():
    torch = pytest.importorskip("torch")
    kv = F.PagedKv(DeviceTensor((4, 8, 16, 64), torch.int8), DeviceTensor((4, 8, 16, 64), torch.int8),
                   DeviceTensor((4, 8), torch.float32), DeviceTensor((4, 8), torch.float32))
    batch = F.PagedBatch(DeviceTensor((2, 2), torch.int32), DeviceTensor((2,), torch.int32))
    k = DeviceTensor((2, 8, 64), torch.float32)
    with pytest.raises(F.FoError, match="positions"):
        F.paged_append(kv, batch, k, k, positions=DeviceTensor((2,), torch.int32), ctx=NoContext)


def test_a_batch_that_another_call_uses_does_not_change_under_it():
    torch = pytest.importorskip("torch")
    batch = F.PagedBatch(DeviceTensor((2, 2), torch.int32), DeviceTensor((2,), torch.int32), rows=9,
                         row_start=DeviceTensor((3,), torch.int32))
    first = batch.of(5)
    second = batch.of(7)
    assert first._obj.total_rows == 5 and second._obj.total_rows == 7
    assert batch.of(7)._obj.total_rows == 7 and batch.of(5)._obj.max_rows == 9


def test_calls_without_rows_need_no_memory():
    """No rows: the rows' pointers may be null (torch gives an empty tensor none); everything else is checked."""
    none, none16, s = rows(data=None), rows(16, data=None, row_stride=1024), spec()
    empty = batch(n_seqs=0, total_rows=0, page_table=None, lens=None)
    calls = [lambda: rope(x=none, out=none, n=0), lambda: append(b=empty, k=none, v=none),
             lambda: append(b=empty, k=none, v=none, q=none16, q_out=none16, s=s),
             lambda: append(b=batch(total_rows=0, max_rows=0), k=none, v=none),
             lambda: attend(b=empty, q=none16, out=none16),
             lambda: attend(b=batch(row_start=BASE, total_rows=0), q=none16, out=none16)]
    for call in calls:
        assert call() == F.ERR_INVALID and last_error() == "null context"
    assert rope(x=none, out=none, n=1) == F.ERR_INVALID and "null pointer" in last_error()
    assert append(b=empty, k=rows(4, data=None), v=none) == F.ERR_INVALID and "cache's heads" in last_error()
