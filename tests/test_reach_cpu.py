"""Refusals, on the host before any device call, of the entry points for
positions on several axes, windows with first positions and shared beginnings;
the layout of what the Python binding packs."""

import ctypes

import pytest

import fo_cuda as F
from test_paged_cpu import BASE, DeviceTensor, batch, last_error, pool, ref, rows

torch = pytest.importorskip("torch")


def axes(**change):
    s = dict(table=BASE, positions=16, row_positions=BASE, row_stride=1, axis_stride=2, rot_dim=64, layout=0, n_axes=3,
             pair_axis=(ctypes.c_uint8 * 128)(*[i % 3 for i in range(128)]))
    s.update(change)
    return F.RopeAxesSpec(*s.values())


def rope(x=rows(), out=rows(), n=2, dim=64, s=axes(), transpose=0):
    return F.lib().fo_rope_by_axes(None, ref(x), ref(out), n, dim, ref(s), transpose)


def append(kv=pool(), b=batch(), k=rows(), v=rows(), q=None, q_out=None, s=axes()):
    return F.lib().fo_paged_append_by_axes(None, ref(kv), ref(b), ref(k), ref(v), ref(q), ref(q_out), ref(s))


def wide(**change):
    return rows(16, **dict(dict(row_stride=1024), **change))


def window(kv=pool(), b=batch(), q=wide(), out=wide(), sinks=None, scale=0.125, window=0, first=0, lse=None):
    return F.lib().fo_paged_window_attention(None, ref(kv), ref(b), ref(q), sinks, scale, window, first, ref(out), lse)


def groups(**change):
    g = dict(seq_start=BASE, lens=BASE, n_groups=1)
    g.update(change)
    return F.PagedPrefixes(*g.values())


def prefix(kv=pool(), b=batch(), g=groups(), q=wide(), out=wide(), sinks=None, scale=0.125, lse=None):
    return F.lib().fo_paged_prefix_attention(None, ref(kv), ref(b), ref(g), ref(q), sinks, scale, ref(out), lse)


ATTENTIONS = [window, prefix]


@pytest.mark.parametrize("call,message", [
    (lambda: rope(s=None), "null axes"),
    (lambda: rope(s=axes(table=None)), "null table"),
    (lambda: rope(s=axes(n_axes=0)), "1 to 4 axes"),
    (lambda: rope(s=axes(n_axes=5)), "1 to 4 axes"),
    (lambda: rope(s=axes(n_axes=2)), "pair 2 has axis 2"),
    (lambda: rope(s=axes(row_positions=None)), "must be given"),
    (lambda: rope(s=axes(row_positions=BASE + 2)), "misaligned positions"),
    (lambda: rope(s=axes(rot_dim=66)), "rot_dim"),
    (lambda: rope(s=axes(layout=2)), "unknown layout"),
    (lambda: rope(out=rows(row_stride=0)), "rows overlap"),
    (lambda: rope(x=rows(dtype=1)), "one type"),
    (lambda: rope(), "null context"),
    (lambda: append(s=None), "null axes"),
    (lambda: append(s=axes(n_axes=1)), "has axis"),
    (lambda: append(k=rows(heads=4)), "cache's heads"),
    (lambda: append(q=rows()), "q needs q_out"),
    (lambda: append(q=rows(), q_out=rows()), "null context"),
    (lambda: append(), "null context"),
    (lambda: window(first=-1), "negative number of first"),
    (lambda: window(window=-1), "negative window"),
    (lambda: prefix(g=None), "null groups"),
    (lambda: prefix(g=groups(n_groups=-1)), "65,535 groups"),
    (lambda: prefix(g=groups(n_groups=65536)), "65,535 groups"),
    (lambda: prefix(g=groups(lens=None)), "null groups' starts"),
    (lambda: prefix(g=groups(seq_start=None)), "null groups' starts"),
    (lambda: prefix(g=groups(lens=BASE + 2)), "misaligned integers"),
    (lambda: prefix(g=groups(seq_start=None, lens=None, n_groups=0)), "null context"),
])
def test_refusals(call, message):
    assert call() == F.ERR_INVALID
    assert message in last_error()


@pytest.mark.parametrize("attention", ATTENTIONS)
@pytest.mark.parametrize("change,message", [
    (dict(kv=None), "null descriptor"), (dict(b=None), "null descriptor"), (dict(q=None), "null pointer"),
    (dict(out=None), "null pointer"), (dict(q=wide(data=None)), "null pointer"), (dict(q=wide(dtype=2)), "unknown type"),
    (dict(q=rows(12, row_stride=1024)), "as many heads"),
    (dict(q=rows(12, row_stride=1024), out=rows(12, row_stride=1024)), "multiple of the KV heads"),
    (dict(q=wide(dtype=1)), "one type"), (dict(scale=float("nan")), "finite"), (dict(lse=BASE + 2), "misaligned"),
    (dict(sinks=BASE + 1), "misaligned"), (dict(out=wide(row_stride=512)), "rows overlap"),
    (dict(kv=pool(page_size=8)), "page_size"), (dict(kv=pool(head_dim=256)), "head_dim must be"),
    (dict(b=batch(n_seqs=0, row_start=BASE, total_rows=5, max_rows=5)), "rows without a sequence"),
    (dict(), "null context"), (dict(b=batch(max_rows=6544, total_rows=13088)), "null context"),
])
def test_attention_refusals(attention, change, message):
    assert attention(**change) == F.ERR_INVALID
    assert message in last_error()


@pytest.mark.parametrize("attention", ATTENTIONS)
def test_too_much_for_32_bits(attention):
    many = batch(n_seqs=60000, total_rows=60000, table_stride=(1 << 31) // 128 - 1)
    assert attention(b=many) == F.ERR_CAPACITY and "2^31 tiles" in last_error()
    many = batch(n_seqs=1, max_rows=1 << 30, total_rows=1 << 30)
    assert attention(b=many, q=rows(32, row_stride=2048), out=rows(32, row_stride=2048)) == F.ERR_CAPACITY
    assert "query rows" in last_error()


def test_python_refusals(monkeypatch):
    table = DeviceTensor((16, 32, 2), torch.float32)
    table.is_contiguous, table.data_ptr, table.get_device = lambda: True, lambda: BASE, lambda: 0
    for bad in ([0] * 31, [0] * 31 + [4], [-1] + [0] * 31):
        with pytest.raises(F.FoError, match="an axis of 0 to 3 for each pair"):
            F.RopeAxes(table, bad)
    rope = F.RopeAxes(table, [0, 2] * 16, "half")
    assert rope.n_axes == 3
    with pytest.raises(F.FoError, match=r"\[axes\]\[rows\]"):
        rope.at(None, 5, 0)
    with pytest.raises(F.FoError, match=r"\[axes\]\[rows\]"):
        rope.at(torch.zeros(2, 5, dtype=torch.int32), 5, 0)
    with pytest.raises(F.FoError, match=r"\[axes\]\[rows\]"):
        rope.at(torch.zeros(3, 4, dtype=torch.int32), 5, 0)
    with pytest.raises(F.FoError, match="CUDA tensor of int32"):
        rope.at(torch.zeros(3, 5, dtype=torch.int32), 5, 0)
    with pytest.raises(F.FoError, match="on GPU 0, the call on GPU 1"):
        rope.at(torch.zeros(3, 5, dtype=torch.int32), 5, 1)
    with pytest.raises(F.FoError, match="one entry more"):
        F.PagedGroups(torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))


def test_packed_axes_are_the_structure():
    packed = F._PACK_AXES(BASE, 16, BASE + 64, 7, 9, 64, 1, 3, bytes([1, 2, 0]))
    assert len(packed) == ctypes.sizeof(F.RopeAxesSpec)
    s = F.RopeAxesSpec.from_buffer_copy(packed)
    assert (s.table, s.positions, s.row_positions, s.row_stride, s.axis_stride) == (BASE, 16, BASE + 64, 7, 9)
    assert (s.rot_dim, s.layout, s.n_axes, list(s.pair_axis[:4])) == (64, 1, 3, [1, 2, 0, 0])
