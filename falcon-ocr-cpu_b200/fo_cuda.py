"""ctypes binding of libfo_cuda.so (include/fo_attention.h), mirroring the
reference's attention operator interface for tests and benchmarks:

* ``attention_with``          kernels::attention_with (src/kernels/attention/mod.rs:256-311)
* ``attention_prefill_bf16``  kernels::attention_prefill_bf16 (mod.rs:321-349)
* ``rope``, ``PagedKv``, ``paged_append``, ``paged_attention``  rotary positions
  and a paged 8-bit cache for many sequences (no counterpart); ``RopeAxes``
  positions on several axes, ``paged_window_attention`` windows with first
  positions and prompts, ``paged_prefix_attention`` shared beginnings; without
  ``ctx`` these run on torch's current stream
* ``SplitPrefix``             quant::kv::SplitPrefix (src/quant/kv.rs:155-972):
  ``from_compact``, ``append``, ``truncate_tail``, ``tail_len``, ``bytes``,
  ``attention_decode``, ``attention_decode_rows``; ``decode_batch`` for pages.

Arrays may be numpy (host memory: the call copies to and from the device) or
CUDA torch tensors (device memory, read and written in place).  Shape errors
raise ``FoError`` as the reference's asserts panic; seal errors raise the
matching subclass as the reference returns an ``anyhow`` error.  There is no
CPU fallback: importing this module without the built library raises.
"""

from __future__ import annotations

import ctypes
import os
import struct
import threading
from typing import Optional, Sequence

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "lib", "libfo_cuda.so")

OK, ERR_INVALID, ERR_PAIR, ERR_NONFINITE, ERR_OVERFLOW, ERR_CAPACITY, ERR_CUDA, ERR_DECLINED = range(8)
MEM_DEVICE, MEM_HOST = 0, 1
KV_F32, KV_Q16, KV_Q8, KV_BF16, KV_Q4 = 0, 1, 2, 3, 4
KV_ROTATED = 16  # flag: blocks stored rotated (src/quant/rotation.rs); with F32, Q8, Q4
KV_Q8_ROT, KV_Q4_ROT = KV_Q8 | KV_ROTATED, KV_Q4 | KV_ROTATED  # Kv::Q8Rot, Kv::Q4Rot
KV_FORMATS = {"f32": KV_F32, "q16": KV_Q16, "q8": KV_Q8, "bf16": KV_BF16, "q4": KV_Q4, "q8r": KV_Q8_ROT,
              "q4r": KV_Q4_ROT, "f32r": KV_F32 | KV_ROTATED}
EXP_EXACT, EXP_FAST = 0, 1
SOFTMAX_ONLINE, SOFTMAX_STATIC = 0, 1


class FoError(RuntimeError):
    status = ERR_INVALID


class PairError(FoError):
    status = ERR_PAIR


class NonFiniteError(FoError):
    status = ERR_NONFINITE


class OverflowKvError(FoError):
    status = ERR_OVERFLOW


class CapacityError(FoError):
    status = ERR_CAPACITY


class CudaError(FoError):
    status = ERR_CUDA


class Declined(FoError):
    status = ERR_DECLINED


_ERRORS = {c.status: c for c in (FoError, PairError, NonFiniteError, OverflowKvError, CapacityError, CudaError,
                                  Declined)}


class Geometry(ctypes.Structure):
    """src/kernels/attention/mod.rs:35-76"""
    _fields_ = [("query_offset", ctypes.c_int64), ("image_start", ctypes.c_int64), ("image_end", ctypes.c_int64)]


class CompactKv(ctypes.Structure):
    """src/kernels/attention/mod.rs:78-97"""
    _fields_ = [("prefix_k", ctypes.c_void_p), ("generated_k", ctypes.c_void_p), ("v", ctypes.c_void_p),
                ("prefix_len", ctypes.c_int64), ("total_len", ctypes.c_int64), ("n_heads", ctypes.c_int64),
                ("n_kv_heads", ctypes.c_int64), ("head_dim", ctypes.c_int64)]


class PrefillOptions(ctypes.Structure):
    """src/kernels/attention/mod.rs:204-221"""
    _fields_ = [("exp", ctypes.c_int32), ("profile", ctypes.c_int32), ("softmax", ctypes.c_int32),
                ("fp32_softmax", ctypes.c_int32)]

    @classmethod
    def exact(cls):
        return cls(EXP_EXACT, 0, SOFTMAX_ONLINE, SOFTMAX_ONLINE)


class Rows(ctypes.Structure):
    """fo_rows: rows of heads in device memory."""
    _fields_ = [("data", ctypes.c_void_p), ("row_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64),
                ("heads", ctypes.c_int32), ("dtype", ctypes.c_int32)]


_PACK_ROWS = struct.Struct("=QqqiI").pack  # Rows and RopeSpec as bytes: a third of a Structure's time
_PACK_ROPE = struct.Struct("=QqQii").pack
_PACK_AXES = struct.Struct("=QqQqqiii128s4x").pack  # RopeAxesSpec


class RopeScaling(ctypes.Structure):
    """fo_rope_scaling"""
    _fields_ = [("theta", ctypes.c_double), ("scaling", ctypes.c_int32), ("factor", ctypes.c_double),
                ("original_positions", ctypes.c_double), ("beta_fast", ctypes.c_double),
                ("beta_slow", ctypes.c_double), ("attention_factor", ctypes.c_double)]


class RopeSpec(ctypes.Structure):
    """fo_rope_spec"""
    _fields_ = [("table", ctypes.c_void_p), ("positions", ctypes.c_int64), ("row_positions", ctypes.c_void_p),
                ("rot_dim", ctypes.c_int32), ("layout", ctypes.c_int32)]


class RopeAxesSpec(ctypes.Structure):
    """fo_rope_axes"""
    _fields_ = [("table", ctypes.c_void_p), ("positions", ctypes.c_int64), ("row_positions", ctypes.c_void_p),
                ("row_stride", ctypes.c_int64), ("axis_stride", ctypes.c_int64), ("rot_dim", ctypes.c_int32),
                ("layout", ctypes.c_int32), ("n_axes", ctypes.c_int32), ("pair_axis", ctypes.c_uint8 * 128)]


class PagedPool(ctypes.Structure):
    """fo_paged_kv"""
    _fields_ = [("k_codes", ctypes.c_void_p), ("v_codes", ctypes.c_void_p), ("k_scales", ctypes.c_void_p),
                ("v_scales", ctypes.c_void_p), ("n_pages", ctypes.c_int64), ("page_size", ctypes.c_int32),
                ("n_kv_heads", ctypes.c_int32), ("head_dim", ctypes.c_int32), ("format", ctypes.c_int32)]


class PagedSequences(ctypes.Structure):
    """fo_paged_batch"""
    _fields_ = [("page_table", ctypes.c_void_p), ("lens", ctypes.c_void_p), ("row_start", ctypes.c_void_p),
                ("table_stride", ctypes.c_int64), ("n_seqs", ctypes.c_int64), ("max_rows", ctypes.c_int64),
                ("total_rows", ctypes.c_int64)]


class PagedPrefixes(ctypes.Structure):
    """fo_paged_groups"""
    _fields_ = [("seq_start", ctypes.c_void_p), ("lens", ctypes.c_void_p), ("n_groups", ctypes.c_int64)]


ROPE_LAYOUTS = {"interleaved": 0, "half": 1}
ROPE_SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3}
PAGED_I8, PAGED_E4M3 = 0, 1

EXPORTS = [
    "fo_version", "fo_last_error", "fo_ctx_create", "fo_ctx_destroy", "fo_ctx_synchronize", "fo_ctx_last_ms",
    "fo_attention", "fo_attention_prefill_bf16", "fo_convert_bf16", "fo_kv_seal", "fo_kv_destroy",
    "fo_kv_set_fast_exp", "fo_kv_append", "fo_kv_truncate_tail", "fo_kv_tail_len", "fo_kv_prefix_len",
    "fo_kv_bytes", "fo_kv_records", "fo_kv_attention_decode", "fo_kv_attention_decode_rows",
    "fo_kv_attention_decode_batch", "fo_kv_append_batch", "fo_qkv_prefix_rows", "fo_kv_append_qkv",
    "fo_sharded_prefill_bf16", "fo_nccl_unique_id", "fo_nccl_comm_init", "fo_nccl_comm_destroy", "fo_kv_seal_layer",
    "fo_kv_plan_create", "fo_kv_plan_step", "fo_kv_plan_finish",
    "fo_decode_rows_static_scratch", "fo_decode_static_scratch_status",
    "fo_selftest_bounded_wait",
    "fo_attention_prefill_bf16_rows", "fo_attention_prefill_bf16_rows_split", "fo_i8_seal", "fo_i8_destroy", "fo_i8_bytes", "fo_i8_records",
    "fo_i8_decode_batch", "fo_draft_kv_create", "fo_draft_kv_destroy", "fo_draft_kv_push", "fo_draft_kv_len",
    "fo_draft_kv_bytes", "fo_draft_kv_records", "fo_draft_attend", "fo_peer_block_register",
    "fo_peer_block_destroy", "fo_sharded_prefill_bf16_peers", "fo_rope_table", "fo_rope", "fo_paged_append",
    "fo_paged_attention", "fo_rope_by_axes", "fo_paged_append_by_axes", "fo_paged_window_attention",
    "fo_paged_prefix_attention",
]

_lib: Optional[ctypes.CDLL] = None


def lib() -> ctypes.CDLL:
    """The loaded library; raises if it was not built (no fallback exists)."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise ImportError(f"{LIB_PATH} is missing: run `python falcon-ocr-cpu_b200/build.py` (no CPU fallback)")
    L = ctypes.CDLL(LIB_PATH)
    P, I32, I64, I = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_int
    PP = ctypes.POINTER(ctypes.c_void_p)
    sigs = {
        "fo_version": (I, []),
        "fo_last_error": (ctypes.c_char_p, []),
        "fo_ctx_create": (I, [I, P, ctypes.POINTER(P)]),
        "fo_ctx_destroy": (I, [P]),
        "fo_ctx_synchronize": (I, [P]),
        "fo_ctx_last_ms": (I, [P, ctypes.POINTER(ctypes.c_float)]),
        "fo_attention": (I, [P, P, ctypes.POINTER(CompactKv), I64, Geometry, P, P, PrefillOptions, I]),
        "fo_attention_prefill_bf16": (I, [P, P, ctypes.POINTER(CompactKv), I64, Geometry, P, P, P, P,
                                          PrefillOptions, I]),
        "fo_convert_bf16": (I, [P, P, P, I64]),
        "fo_kv_seal": (I, [P, P, P, I64, I64, I64, I64, I64, I32, I32, I, ctypes.POINTER(P)]),
        "fo_kv_destroy": (I, [P]),
        "fo_kv_set_fast_exp": (I, [P, I32]),
        "fo_kv_append": (I, [P, P, P, I64, I]),
        "fo_kv_truncate_tail": (I, [P, I64]),
        "fo_kv_tail_len": (I64, [P]),
        "fo_kv_prefix_len": (I64, [P]),
        "fo_kv_bytes": (I64, [P]),
        "fo_kv_records": (I, [P, PP, PP, PP, PP, ctypes.POINTER(I64), ctypes.POINTER(I64)]),
        "fo_kv_attention_decode": (I, [P, P, I64, P, P, I]),
        "fo_kv_attention_decode_rows": (I, [P, P, I64, P, P, I]),
        "fo_kv_attention_decode_batch": (I, [PP, I64, PP, PP, PP]),
        "fo_kv_append_batch": (I, [PP, I64, PP, PP, I64]),
        "fo_qkv_prefix_rows": (I, [P, P, P, I64, I64, I64, P, P, P, P, P]),
        "fo_kv_append_qkv": (I, [P, P, P, I64, P]),
        "fo_sharded_prefill_bf16": (I, [P, P, I32, I32, P, P, P, I64, I64, I64, Geometry, P, PrefillOptions, I32,
                                        I32, P]),
        "fo_nccl_unique_id": (I, [P]),
        "fo_nccl_comm_init": (I, [P, I32, I32, P, ctypes.POINTER(P)]),
        "fo_nccl_comm_destroy": (I, [P]),
        "fo_kv_plan_create": (I, [PP, I64, PP, PP, PP, PP, PP, ctypes.POINTER(P)]),
        "fo_kv_plan_step": (I, [P]),
        "fo_kv_plan_finish": (I, [P]),
        "fo_kv_seal_layer": (I, [P, I32, ctypes.c_uint64, I32, I32, I32, P, P, I64, I64, I64, I64, I64, I32,
                                 ctypes.POINTER(P)]),
        "fo_decode_rows_static_scratch": (I, [P, P, P, P, I32, I64, I64, I64, I64, I64, I64, P, I64, P, I32, P, P]),
        "fo_decode_static_scratch_status": (I, [P]),
        "fo_selftest_bounded_wait": (I, [P, ctypes.c_uint64]),
        "fo_attention_prefill_bf16_rows": (I, [P, P, P, P, I64, I64, I64, Geometry, P, P, I64, I64, PrefillOptions]),
        "fo_attention_prefill_bf16_rows_split": (I, [P, P, P, P, I64, I64, I64, Geometry, P, P, I32, I64, I64,
                                                     PrefillOptions, I]),
        "fo_i8_seal": (I, [P, P, P, I64, I64, I, ctypes.POINTER(P)]),
        "fo_i8_destroy": (I, [P]),
        "fo_i8_bytes": (I64, [P]),
        "fo_i8_records": (I, [P, PP, PP, PP, PP]),
        "fo_i8_decode_batch": (I, [PP, I64, PP, PP, PP, I32]),
        "fo_draft_kv_create": (I, [P, I64, ctypes.POINTER(P)]),
        "fo_draft_kv_destroy": (I, [P]),
        "fo_draft_kv_push": (I, [P, P, P, I64, I]),
        "fo_draft_kv_len": (I64, [P]),
        "fo_draft_kv_bytes": (I64, [P]),
        "fo_draft_kv_records": (I, [P, PP, PP, PP, PP]),
        "fo_draft_attend": (I, [P, P, I64, I64, P, P, I64, P, I]),
        "fo_peer_block_register": (I, [P, P, I32, I32, P, I64, ctypes.POINTER(P)]),
        "fo_peer_block_destroy": (I, [P]),
        "fo_sharded_prefill_bf16_peers": (I, [P, P, P, P, P, I64, I64, I64, Geometry, P, PrefillOptions, I32]),
        "fo_rope_table": (I, [P, P, I64, I32, RopeScaling]),
        "fo_rope": (I, [P, P, P, I64, I32, P, I32]),
        "fo_paged_append": (I, [P, P, P, P, P, P, P, P]),
        "fo_paged_attention": (I, [P, P, P, P, P, ctypes.c_float, I64, P, P]),
        "fo_rope_by_axes": (I, [P, P, P, I64, I32, P, I32]),
        "fo_paged_append_by_axes": (I, [P, P, P, P, P, P, P, P]),
        "fo_paged_window_attention": (I, [P, P, P, P, P, ctypes.c_float, I64, I64, P, P]),
        "fo_paged_prefix_attention": (I, [P, P, P, P, P, P, ctypes.c_float, P, P]),
    }
    for name, (res, args) in sigs.items():
        fn = getattr(L, name)
        fn.restype = res
        fn.argtypes = args
    _lib = L
    return L


def check(status: int) -> None:
    if status != OK:
        msg = lib().fo_last_error().decode(errors="replace")
        raise _ERRORS.get(status, FoError)(f"fo status {status}: {msg}")


def _is_torch(x) -> bool:
    return type(x).__module__.startswith("torch")


def _on_device(a) -> bool:
    return _is_torch(a) and a.is_cuda


def _ptr_mem(arrays):
    """Pointers of a call's arrays and its memory mode: all host (numpy
    arrays or CPU torch tensors, e.g. pinned) or all device (CUDA tensors)."""
    kinds = {_on_device(a) for a in arrays if a is not None}
    if len(kinds) > 1:
        raise FoError("mix of host and device arrays in one call")
    device = kinds == {True}
    ptrs = []
    for a in arrays:
        if a is None:
            ptrs.append(None)
        elif _is_torch(a):
            if not a.is_contiguous():
                raise FoError("arrays must be contiguous")
            ptrs.append(a.data_ptr())
        else:
            if not (a.flags["C_CONTIGUOUS"]):
                raise FoError("host arrays must be C-contiguous")
            ptrs.append(a.ctypes.data)
    return ptrs, (MEM_DEVICE if device else MEM_HOST)


def _f32(a):
    if a is None or _is_torch(a):
        return a
    return np.ascontiguousarray(a, dtype=np.float32)


class Context:
    """A device and a stream (fo_ctx)."""

    def __init__(self, device: int = 0, stream: Optional[int] = None):
        h = ctypes.c_void_p()
        check(lib().fo_ctx_create(device, stream, ctypes.byref(h)))
        self.handle = h
        self.device = device

    def close(self):
        if self.handle:
            lib().fo_ctx_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def synchronize(self):
        check(lib().fo_ctx_synchronize(self.handle))

    def last_ms(self) -> float:
        v = ctypes.c_float()
        check(lib().fo_ctx_last_ms(self.handle, ctypes.byref(v)))
        return v.value

    def selftest_bounded_wait(self, limit_ns: int) -> int:
        """fo_selftest_bounded_wait: the raw status (FO_ERR_CUDA when the
        device wait gave up after limit_ns, as designed)."""
        return lib().fo_selftest_bounded_wait(self.handle, limit_ns)


_default: Optional[Context] = None


def default_context() -> Context:
    global _default
    if _default is None:
        _default = Context(0)
    return _default


def attention_with(q, prefix_k, v, query_len, geometry, sinks, output, n_heads, n_kv_heads, head_dim,
                   generated_k=None, prefix_len=None, total_len=None, options=None, ctx=None):
    """kernels::attention_with: `output` is overwritten."""
    ctx = ctx or default_context()
    q, prefix_k, v, sinks, generated_k = _f32(q), _f32(prefix_k), _f32(v), _f32(sinks), _f32(generated_k)
    (pq, ppk, pgk, pv, ps, po), mem = _ptr_mem([q, prefix_k, generated_k, v, sinks, output])
    if prefix_len is None:
        prefix_len = prefix_k.numel() // (n_heads * head_dim) if _is_torch(prefix_k) else prefix_k.size // (
            n_heads * head_dim)
    if total_len is None:
        total_len = (v.numel() if _is_torch(v) else v.size) // (n_kv_heads * head_dim)
    kv = CompactKv(ppk, pgk, pv, prefix_len, total_len, n_heads, n_kv_heads, head_dim)
    g = Geometry(*geometry)
    check(lib().fo_attention(ctx.handle, pq, ctypes.byref(kv), query_len, g, ps, po, options or PrefillOptions.exact(),
                             mem))
    return output


def attention_prefill_bf16(q, k, v, geometry, sinks, output, n_heads, n_kv_heads, keys_bf16=None, values_bf16=None,
                           options=None, ctx=None):
    """kernels::attention_prefill_bf16 over a pure prefix; raises Declined for other shapes."""
    ctx = ctx or default_context()
    q, k, v, sinks = _f32(q), _f32(k), _f32(v), _f32(sinks)
    (pq, pk, pv, ps, po), mem = _ptr_mem([q, k, v, sinks, output])
    total = (q.numel() if _is_torch(q) else q.size) // (n_heads * 64)
    kv = CompactKv(pk, None, pv, total, total, n_heads, n_kv_heads, 64)
    kb = keys_bf16.data_ptr() if keys_bf16 is not None else None
    vb = values_bf16.data_ptr() if values_bf16 is not None else None
    if options is None:
        options = PrefillOptions(EXP_FAST, 0, SOFTMAX_STATIC, SOFTMAX_ONLINE)
    check(lib().fo_attention_prefill_bf16(ctx.handle, pq, ctypes.byref(kv), total, Geometry(*geometry), ps, po, kb, vb,
                                          options, mem))
    return output


def attention_prefill_bf16_rows(q, keys_bf16, values_bf16, geometry, sinks, output, n_heads, n_kv_heads, query_begin,
                                query_end, options=None, ctx=None, kv_splits=1):
    """fo_attention_prefill_bf16_rows: the BF16 prefill of query rows
    [query_begin, query_end) of a pure prefix (CUDA tensors; BF16 keys and
    values already converted).  Rows outside the range are left as they are.
    kv_splits > 1 cuts each query pair's keys into that many ranges, and a
    BF16 `output` takes the rounded result directly
    (fo_attention_prefill_bf16_rows_split)."""
    ctx = ctx or default_context()
    for a in (q, keys_bf16, values_bf16, sinks, output):
        if not _on_device(a) or not a.is_contiguous():
            raise FoError("fo_attention_prefill_bf16_rows takes contiguous CUDA tensors")
    total = q.numel() // (n_heads * 64)
    if options is None:
        options = PrefillOptions(EXP_FAST, 0, SOFTMAX_STATIC, SOFTMAX_ONLINE)
    out_bf16 = 1 if str(output.dtype) == "torch.bfloat16" else 0
    if kv_splits == 1 and not out_bf16:
        check(lib().fo_attention_prefill_bf16_rows(ctx.handle, q.data_ptr(), keys_bf16.data_ptr(),
                                                   values_bf16.data_ptr(), total, n_heads, n_kv_heads,
                                                   Geometry(*geometry), sinks.data_ptr(), output.data_ptr(),
                                                   query_begin, query_end, options))
    else:
        check(lib().fo_attention_prefill_bf16_rows_split(ctx.handle, q.data_ptr(), keys_bf16.data_ptr(),
                                                         values_bf16.data_ptr(), total, n_heads, n_kv_heads,
                                                         Geometry(*geometry), sinks.data_ptr(), output.data_ptr(),
                                                         out_bf16, query_begin, query_end, options, kv_splits))
    return output


class SplitPrefix:
    """quant::kv::SplitPrefix on the device (src/quant/kv.rs:155-972)."""

    def __init__(self, handle, ctx, heads):
        self.handle = handle
        self.ctx = ctx
        self.heads = heads

    @classmethod
    def from_compact(cls, k, v, prefix_len, capacity, fmt="f32", heads=16, kv_heads=8, head_dim=64, chunks=0,
                     ctx=None):
        ctx = ctx or default_context()
        fmt = KV_FORMATS[fmt] if isinstance(fmt, str) else fmt
        k, v = _f32(k), _f32(v)
        (pk, pv), mem = _ptr_mem([k, v])
        h = ctypes.c_void_p()
        check(lib().fo_kv_seal(ctx.handle, pk, pv, prefix_len, capacity, heads, kv_heads, head_dim, fmt, chunks, mem,
                               ctypes.byref(h)))
        return cls(h, ctx, heads)

    @classmethod
    def seal_layer(cls, layer, k, v, filled, prefix_len, capacity, mode="bf16", kv_q8_layers=0, fast_exps=False,
                   decode_fast_exp=None, heads=16, kv_heads=8, chunks=0, ctx=None):
        """fo_kv_seal_layer (model::cache::seal_layer, src/model/cache.rs:218-276)
        on device tensors k, v: Q8 records where bit `layer` of kv_q8_layers is
        set, `mode` otherwise."""
        ctx = ctx or default_context()
        mode = KV_FORMATS[mode] if isinstance(mode, str) else mode
        req = -1 if decode_fast_exp is None else int(bool(decode_fast_exp))
        h = ctypes.c_void_p()
        check(lib().fo_kv_seal_layer(ctx.handle, layer, kv_q8_layers, mode, int(bool(fast_exps)), req, k.data_ptr(),
                                     v.data_ptr(), filled, prefix_len, capacity, heads, kv_heads, chunks,
                                     ctypes.byref(h)))
        return cls(h, ctx, heads)

    def close(self):
        if self.handle:
            lib().fo_kv_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def with_fast_exp(self, fast: bool = True) -> "SplitPrefix":
        check(lib().fo_kv_set_fast_exp(self.handle, int(bool(fast))))
        return self

    def append(self, k, v):
        k, v = _f32(k), _f32(v)
        (pk, pv), mem = _ptr_mem([k, v])
        n = (k.numel() if _is_torch(k) else k.size) // (self.heads * 64)
        check(lib().fo_kv_append(self.handle, pk, pv, n, mem))

    def truncate_tail(self, tail_len: int):
        check(lib().fo_kv_truncate_tail(self.handle, tail_len))

    @property
    def tail_len(self) -> int:
        return int(lib().fo_kv_tail_len(self.handle))

    @property
    def prefix_len(self) -> int:
        return int(lib().fo_kv_prefix_len(self.handle))

    def bytes(self) -> int:
        return int(lib().fo_kv_bytes(self.handle))

    def records(self):
        """(codes, scales, tail_codes, tail_scales) device pointers and strides."""
        ptrs = [ctypes.c_void_p() for _ in range(4)]
        ps, ts = ctypes.c_int64(), ctypes.c_int64()
        check(lib().fo_kv_records(self.handle, *[ctypes.byref(p) for p in ptrs], ctypes.byref(ps), ctypes.byref(ts)))
        return [p.value for p in ptrs], ps.value, ts.value

    def attention_decode(self, q, total_len, sinks, output):
        q, sinks = _f32(q), _f32(sinks)
        (pq, ps, po), mem = _ptr_mem([q, sinks, output])
        check(lib().fo_kv_attention_decode(self.handle, pq, total_len, ps, po, mem))
        return output

    def attention_decode_rows(self, q, rows, sinks, output):
        q, sinks = _f32(q), _f32(sinks)
        (pq, ps, po), mem = _ptr_mem([q, sinks, output])
        check(lib().fo_kv_attention_decode_rows(self.handle, pq, rows, ps, po, mem))
        return output


def decode_batch(caches: Sequence[SplitPrefix], qs, sinks, outputs):
    """One single-row decode per page in one launch (device tensors)."""
    n = len(caches)
    arr = lambda xs: (ctypes.c_void_p * n)(*xs)  # noqa: E731
    check(lib().fo_kv_attention_decode_batch(arr([c.handle.value for c in caches]), n, arr([q.data_ptr() for q in qs]),
                                             arr([s.data_ptr() for s in sinks]),
                                             arr([o.data_ptr() for o in outputs])))


def append_batch(caches: Sequence[SplitPrefix], ks, vs, rows: int):
    """fo_kv_append_batch: `rows` expanded rows into each cache in one launch
    (device tensors ks[i], vs[i] of [rows][heads][64])."""
    n = len(caches)
    arr = lambda xs: (ctypes.c_void_p * n)(*xs)  # noqa: E731
    check(lib().fo_kv_append_batch(arr([c.handle.value for c in caches]), n, arr([k.data_ptr() for k in ks]),
                                   arr([v.data_ptr() for v in vs]), rows))


def qkv_prefix_rows(qkv, rope, rows: int, q, k, v, k_bf16=None, v_bf16=None, heads: int = 16, kv_heads: int = 8,
                    ctx=None):
    """fo_qkv_prefix_rows on device tensors: the fused split + per-head RMS
    norm + RoPE of projection rows into q, k (and their BF16 copies)."""
    ctx = ctx or default_context()
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    check(lib().fo_qkv_prefix_rows(ctx.handle, qkv.data_ptr(), rope.data_ptr(), rows, heads, kv_heads, q.data_ptr(),
                                   k.data_ptr(), v.data_ptr(), ptr(k_bf16), ptr(v_bf16)))


def append_qkv(cache: SplitPrefix, qkv, rope, rows: int, q):
    """fo_kv_append_qkv on device tensors: decode rows' queries into q, their
    keys and values appended to the cache's tail."""
    check(lib().fo_kv_append_qkv(cache.handle, qkv.data_ptr(), rope.data_ptr(), rows, q.data_ptr()))


class BatchPlan:
    """fo_kv_plan_*: the append of one row and the one-row decode of every
    cache as one device-resident step (graph-capturable).  ks, vs, qs, sinks
    and outs are device tensors the plan reads and writes at every step."""

    def __init__(self, caches, ks, vs, qs, sinks, outs):
        n = len(caches)
        arr = lambda xs: (ctypes.c_void_p * n)(*xs)  # noqa: E731
        h = ctypes.c_void_p()
        check(lib().fo_kv_plan_create(arr([c.handle.value for c in caches]), n, arr([t.data_ptr() for t in ks]),
                                      arr([t.data_ptr() for t in vs]), arr([t.data_ptr() for t in qs]),
                                      arr([t.data_ptr() for t in sinks]), arr([t.data_ptr() for t in outs]),
                                      ctypes.byref(h)))
        self.handle = h
        self._keep = (ks, vs, qs, sinks, outs)

    def step(self):
        check(lib().fo_kv_plan_step(self.handle))

    def finish(self):
        if self.handle:
            h, self.handle = self.handle, None
            check(lib().fo_kv_plan_finish(h))


class NcclComm:
    """An NCCL communicator from the library's NCCL (fo_nccl_comm_init); rank 0
    makes the id with nccl_unique_id() and the caller shares it."""

    def __init__(self, world: int, rank: int, uid: bytes, ctx=None):
        ctx = ctx or default_context()
        if len(uid) != 128:
            raise FoError("an NCCL unique id is 128 bytes")
        buf = (ctypes.c_uint8 * 128).from_buffer_copy(uid)
        h = ctypes.c_void_p()
        check(lib().fo_nccl_comm_init(ctx.handle, world, rank, buf, ctypes.byref(h)))
        self.handle, self.world, self.rank = h, world, rank

    def close(self):
        if self.handle:
            check(lib().fo_nccl_comm_destroy(self.handle))
            self.handle = None


def nccl_unique_id() -> bytes:
    buf = (ctypes.c_uint8 * 128)()
    check(lib().fo_nccl_unique_id(buf))
    return bytes(buf)


def sharded_prefill_bf16(comm: NcclComm, q, keys_bf16, values_bf16, geometry, sinks, gathered, n_heads, n_kv_heads,
                         n_bands=1, kv_splits=0, options=None, ctx=None):
    """fo_sharded_prefill_bf16 on this rank's heads (contiguous CUDA tensors);
    `gathered` BF16 holds the bands' rank-major blocks one after another."""
    ctx = ctx or default_context()
    total = q.numel() // (n_heads * 64)
    if options is None:
        options = PrefillOptions(EXP_FAST, 0, SOFTMAX_STATIC, SOFTMAX_ONLINE)
    check(lib().fo_sharded_prefill_bf16(ctx.handle, comm.handle, comm.rank, comm.world, q.data_ptr(),
                                        keys_bf16.data_ptr(), values_bf16.data_ptr(), total, n_heads, n_kv_heads,
                                        Geometry(*geometry), sinks.data_ptr(), options, n_bands, kv_splits,
                                        gathered.data_ptr()))
    return gathered


class DraftKv:
    """The draft head's int8 key/value cache on the device (fo_draft_kv_*:
    DraftState's Kv::Q8 and attend, src/draft_head.rs:177-220, 548-759)."""

    def __init__(self, capacity, ctx=None):
        ctx = ctx or default_context()
        h = ctypes.c_void_p()
        check(lib().fo_draft_kv_create(ctx.handle, capacity, ctypes.byref(h)))
        self.handle, self.capacity, self.ctx = h, capacity, ctx

    @property
    def len(self) -> int:
        return lib().fo_draft_kv_len(self.handle)

    def push(self, keys, values):
        """Rows [rows][512] of keys and values (numpy: host; CUDA tensors: device)."""
        keys, values = _f32(keys), _f32(values)
        (pk, pv), mem = _ptr_mem([keys, values])
        n = keys.numel() if _is_torch(keys) else keys.size
        check(lib().fo_draft_kv_push(self.handle, pk, pv, n // 512, mem))

    def attend(self, q, bases, output, window=0, chain_keys=None, chain_values=None):
        """Attention of q [16][64] over the verified rows (the newest `window`
        of the first `bases`; 0: all) and the chain rows [chain][512]."""
        chain = 0
        if chain_keys is not None:
            chain = (chain_keys.numel() if _is_torch(chain_keys) else np.asarray(chain_keys).size) // 512
        q = _f32(q)
        ck = _f32(chain_keys) if chain else None
        cv = _f32(chain_values) if chain else None
        (pq, pk, pv, po), mem = _ptr_mem([q, ck, cv, output])
        check(lib().fo_draft_attend(self.handle, pq, bases, window, pk, pv, chain, po, mem))
        return output

    def records(self):
        """Device pointers (key_codes, key_scales, value_codes, value_scales)."""
        ptrs = [ctypes.c_void_p() for _ in range(4)]
        check(lib().fo_draft_kv_records(self.handle, *[ctypes.byref(p) for p in ptrs]))
        return tuple(p.value for p in ptrs)

    def close(self):
        if self.handle:
            lib().fo_draft_kv_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class PeerBlock:
    """fo_peer_block_register: every rank's gathered buffer mapped into this
    process (collective over the communicator's ranks)."""

    def __init__(self, comm: "NcclComm", gathered, ctx=None):
        ctx = ctx or default_context()
        h = ctypes.c_void_p()
        nbytes = gathered.numel() * gathered.element_size()
        check(lib().fo_peer_block_register(ctx.handle, comm.handle, comm.rank, comm.world, gathered.data_ptr(), nbytes,
                                           ctypes.byref(h)))
        self.handle, self.gathered = h, gathered

    def close(self):
        if self.handle:
            lib().fo_peer_block_destroy(self.handle)
            self.handle = None


def sharded_prefill_bf16_peers(block: PeerBlock, q, keys_bf16, values_bf16, geometry, sinks, n_heads, n_kv_heads,
                               kv_splits=0, options=None, ctx=None):
    """fo_sharded_prefill_bf16_peers: this rank's heads, every finished row
    stored by the kernels into all ranks' registered blocks."""
    ctx = ctx or default_context()
    total = q.numel() // (n_heads * 64)
    if options is None:
        options = PrefillOptions(EXP_FAST, 0, SOFTMAX_STATIC, SOFTMAX_ONLINE)
    check(lib().fo_sharded_prefill_bf16_peers(ctx.handle, block.handle, q.data_ptr(), keys_bf16.data_ptr(),
                                              values_bf16.data_ptr(), total, n_heads, n_kv_heads, Geometry(*geometry),
                                              sinks.data_ptr(), options, kv_splits))
    return block.gathered


class Int8Cache:
    """BASELINE config 4's INT8 KV format on the device (fo_i8_seal): keys
    and values [len][heads][64] quantized per (head, 64-position group)."""

    def __init__(self, k, v, heads=16, ctx=None):
        ctx = ctx or default_context()
        k, v = _f32(k), _f32(v)
        (pk, pv), mem = _ptr_mem([k, v])
        n = k.numel() if _is_torch(k) else k.size
        self.len, self.heads, self.ctx = n // (heads * 64), heads, ctx
        h = ctypes.c_void_p()
        check(lib().fo_i8_seal(ctx.handle, pk, pv, self.len, heads, mem, ctypes.byref(h)))
        self.handle = h

    def bytes(self) -> int:
        return lib().fo_i8_bytes(self.handle)

    def records(self):
        """Device pointers (k_codes, k_scales, v_codes, v_scales)."""
        ptrs = [ctypes.c_void_p() for _ in range(4)]
        check(lib().fo_i8_records(self.handle, *[ctypes.byref(p) for p in ptrs]))
        return tuple(p.value for p in ptrs)

    def close(self):
        if self.handle:
            lib().fo_i8_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def int8_decode_batch(caches: Sequence[Int8Cache], qs, sinks, outputs, fast_exp=False):
    """One decode row per page in one launch (CUDA tensors)."""
    n = len(caches)
    arr = lambda xs: (ctypes.c_void_p * n)(*xs)  # noqa: E731
    check(lib().fo_i8_decode_batch(arr([c.handle.value for c in caches]), n, arr([q.data_ptr() for q in qs]),
                                   arr([s.data_ptr() for s in sinks]), arr([o.data_ptr() for o in outputs]),
                                   int(bool(fast_exp))))


def decode_rows_static_scratch(cache: SplitPrefix, fmt, q, rows, sinks, output, fast_exp=False, stream=None):
    """fo_decode_rows_static_scratch over a sealed cache's records: the decode
    for callers that cannot allocate device memory (q, sinks and output are
    CUDA tensors; the partials live in the library's static array)."""
    fmt = KV_FORMATS[fmt] if isinstance(fmt, str) else fmt
    (codes, scales, tcodes, tscales), ps, ts = cache.records()
    check(lib().fo_decode_rows_static_scratch(codes, scales, tcodes, tscales, fmt, cache.prefix_len, ps,
                                              cache.tail_len, ts, cache.heads, cache.heads // 2, q.data_ptr(), rows,
                                              sinks.data_ptr(), int(bool(fast_exp)), output.data_ptr(), stream))
    return output


def static_scratch_status(stream=None):
    """fo_decode_static_scratch_status: raises CudaError if a bounded device
    wait of a static-scratch decode gave up since the last check."""
    check(lib().fo_decode_static_scratch_status(stream))


# ------------------------------------------------ rotary positions, paged cache
_ROW_TYPES = None  # torch dtype -> FO_DT_*
_stream_contexts = {}
_stream_contexts_lock = threading.Lock()


def _torch():
    global _ROW_TYPES
    import torch
    if _ROW_TYPES is None:
        _ROW_TYPES = {torch.float32: 0, torch.bfloat16: 1}
    return torch


def stream_context(device: int) -> Context:
    """The context of torch's current stream on `device`, made at its first
    use.  That and the first attention on it allocate, which a capture refuses:
    a graph is captured on a stream that its calls have run on before
    (``torch.cuda.graph(g, stream=side)``; without ``stream`` torch captures on
    one of its own).  Attentions of one context share its scratch: graphs that
    were captured on one stream must not be replayed at the same time."""
    stream = _torch()._C._cuda_getCurrentRawStream(device)
    ctx = _stream_contexts.get((device, stream))
    if ctx is None:
        with _stream_contexts_lock:  # one for all threads on the stream
            ctx = _stream_contexts.get((device, stream))
            if ctx is None:
                ctx = _stream_contexts[(device, stream)] = Context(device, stream or None)
    return ctx


def _rows(t, name: str, device: int) -> bytes:
    """A tensor [rows][heads][head_dim] on GPU `device` as fo_rows; rows and
    heads in any strides."""
    if _ROW_TYPES is None:
        _torch()
    kind, at = _ROW_TYPES.get(t.dtype), t.get_device()
    if kind is None or at < 0 or t.dim() != 3:
        raise FoError(f"{name} must be a CUDA tensor [rows][heads][head_dim] of float32 or bfloat16")
    if at != device:
        raise FoError(f"{name} is on GPU {at}, the call on GPU {device}")
    row, head, one = t.stride()
    if one != 1:
        raise FoError(f"{name}: a head's values must be adjacent")
    return _PACK_ROWS(t.data_ptr(), row, head, t.size(1), kind)


def _device_ints(t, name: str, device: int):
    if not t.is_cuda or not t.is_contiguous() or t.dtype != _torch().int32:
        raise FoError(f"{name} must be a contiguous CUDA tensor of int32")
    if t.get_device() != device:
        raise FoError(f"{name} is on GPU {t.get_device()}, the call on GPU {device}")
    return t.data_ptr()


def _floats(t, n: int, name: str, device: int):
    if not t.is_cuda or not t.is_contiguous() or t.numel() != n or t.dtype != _torch().float32:
        raise FoError(f"{name} must be a contiguous CUDA tensor of {n} float32")
    if t.get_device() != device:
        raise FoError(f"{name} is on GPU {t.get_device()}, the call on GPU {device}")
    return t.data_ptr()


def _context(ctx, device: int):
    if ctx is None:
        return stream_context(device)
    if ctx.device != device:
        raise FoError(f"the context is on GPU {ctx.device}, the call's tensors on GPU {device}")
    return ctx


def rope_table(table, theta=10000.0, scaling="none", factor=1.0, original_positions=0, beta_fast=32.0, beta_slow=1.0,
               attention_factor=0.0, ctx=None):
    """fo_rope_table: fills the CUDA tensor `table` [positions][rot_dim / 2][2]
    with {cos, sin}; scaling "none", "linear", "ntk" or "yarn"."""
    if not _on_device(table) or not table.is_contiguous() or table.dim() != 3 or table.shape[2] != 2 or \
            str(table.dtype) != "torch.float32":
        raise FoError("a rope table is a contiguous float32 CUDA tensor [positions][rot_dim / 2][2]")
    ctx = _context(ctx, table.get_device())
    check(lib().fo_rope_table(ctx.handle, table.data_ptr(), table.shape[0], 2 * table.shape[1],
                              RopeScaling(theta, ROPE_SCALINGS[scaling], factor, original_positions, beta_fast,
                                          beta_slow, attention_factor)))
    return table


class Rope:
    """A rope table and the layout of the pairs that it turns."""

    rope_call, append_call = "fo_rope", "fo_paged_append"

    def __init__(self, table, layout="interleaved"):
        if not _on_device(table) or not table.is_contiguous() or table.dim() != 3 or table.shape[2] != 2 or \
                str(table.dtype) != "torch.float32":
            raise FoError("a rope table is a contiguous float32 CUDA tensor [positions][rot_dim / 2][2]")
        self.table, self.device = table, table.get_device()
        self.spec = (table.data_ptr(), table.shape[0], 2 * table.shape[1], ROPE_LAYOUTS[layout])
        self.plain = _PACK_ROPE(self.spec[0], self.spec[1], 0, self.spec[2], self.spec[3])

    def at(self, positions, rows: int, device: int) -> bytes:
        if self.device != device:
            raise FoError(f"the rope table is on GPU {self.device}, the call on GPU {device}")
        if positions is None:
            return self.plain
        if positions.numel() != rows:
            raise FoError("one position for each row")
        table, n, rot_dim, layout = self.spec
        return _PACK_ROPE(table, n, _device_ints(positions, "positions", device), rot_dim, layout)


class RopeAxes(Rope):
    """A rope table whose pairs turn by positions on several axes (time, height
    and width, say): `axes` names each of the rot_dim / 2 pairs' axis, 0 to 3.
    Calls with it want `positions` [axes][rows] int32, in any strides."""

    rope_call, append_call = "fo_rope_by_axes", "fo_paged_append_by_axes"

    def __init__(self, table, axes, layout="interleaved"):
        super().__init__(table, layout)
        axes = [int(a) for a in axes]
        if len(axes) != table.shape[1] or len(axes) > 128 or min(axes) < 0 or max(axes) > 3:
            raise FoError("rope axes: an axis of 0 to 3 for each pair of the table, 128 pairs at most")
        self.n_axes, self.pair_axis = max(axes) + 1, bytes(axes)

    def at(self, positions, rows: int, device: int) -> bytes:
        if self.device != device:
            raise FoError(f"the rope table is on GPU {self.device}, the call on GPU {device}")
        if positions is None or positions.dim() != 2 or positions.shape[0] < self.n_axes or positions.shape[1] != rows:
            raise FoError("positions on axes must be [axes][rows]")
        if not positions.is_cuda or positions.dtype != _torch().int32:
            raise FoError("positions must be a CUDA tensor of int32")
        if positions.get_device() != device:
            raise FoError(f"positions is on GPU {positions.get_device()}, the call on GPU {device}")
        table, n, rot_dim, layout = self.spec
        axis_stride, row_stride = positions.stride()
        return _PACK_AXES(table, n, positions.data_ptr(), row_stride, axis_stride, rot_dim, layout, self.n_axes,
                          self.pair_axis)


def rope(x, out, rope: Rope, positions=None, inverse=False, ctx=None):
    """fo_rope: rows x [rows][heads][head_dim] rotated into `out` (x itself is
    allowed) at `positions` [rows] int32 (None: the row's number), or with a
    RopeAxes (fo_rope_by_axes) at `positions` [axes][rows].  inverse: the
    transposed rotation, which takes a gradient back."""
    device = x.get_device()
    a, b = _rows(x, "x", device), _rows(out, "out", device)
    shape = x.shape
    if shape != out.shape:
        raise FoError("rope: x and out must have one shape")
    rows, _, dim = shape
    ctx = _context(ctx, device)
    call = getattr(lib(), rope.rope_call)
    check(call(ctx.handle, a, b, rows, dim, rope.at(positions, rows, device), 1 if inverse else 0))
    return out


class PagedKv:
    """The pool of a paged 8-bit cache (fo_paged_kv): codes [pages][kv heads]
    [page size][head dim] of int8 or float8_e4m3fn, scales [pages][kv heads]
    float32, all contiguous CUDA tensors of the caller's."""

    def __init__(self, k_codes, v_codes, k_scales, v_scales):
        torch = _torch()
        formats = {torch.int8: PAGED_I8, torch.float8_e4m3fn: PAGED_E4M3}
        if k_codes.dtype not in formats or v_codes.dtype != k_codes.dtype:
            raise FoError("paged codes must be int8 or float8_e4m3fn, keys and values alike")
        if k_codes.dim() != 4 or k_codes.shape != v_codes.shape:
            raise FoError("paged codes must be [pages][kv heads][page size][head dim], keys and values alike")
        for t in (k_scales, v_scales):
            if t.dtype != torch.float32 or t.shape != k_codes.shape[:2]:
                raise FoError("paged scales must be float32 [pages][kv heads]")
        for t in (k_codes, v_codes, k_scales, v_scales):
            if not t.is_cuda or not t.is_contiguous():
                raise FoError("paged codes and scales must be contiguous CUDA tensors")
            if t.get_device() != k_codes.get_device():
                raise FoError("paged codes and scales must be on one GPU")
        self.keep = (k_codes, v_codes, k_scales, v_scales)
        n_pages, kv_heads, page_size, self.head_dim = k_codes.shape
        self.device = k_codes.get_device()
        self.pool = PagedPool(k_codes.data_ptr(), v_codes.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(),
                              n_pages, page_size, kv_heads, self.head_dim, formats[k_codes.dtype])
        self.ref, self.scale = ctypes.byref(self.pool), self.head_dim ** -0.5


class PagedBatch:
    """The sequences of paged calls (fo_paged_batch): page_table [seqs][pages]
    and lens [seqs] int32, lens counting the call's rows; `rows` of each
    sequence, or at most, with row_start [seqs + 1] int32, as many as that
    says.  The tensors are the caller's and may change between calls."""

    def __init__(self, page_table, lens, rows=1, row_start=None):
        if page_table.dim() != 2 or page_table.shape[0] != lens.numel():
            raise FoError("page_table must be [seqs][pages], with one length for each")
        if row_start is not None and row_start.numel() != lens.numel() + 1:
            raise FoError("row_start must have one entry more than there are sequences")
        self.keep = (page_table, lens, row_start)
        n = lens.numel()
        self.device = device = page_table.get_device()
        self.sequences = PagedSequences(
            _device_ints(page_table, "page_table", device), _device_ints(lens, "lens", device),
            None if row_start is None else _device_ints(row_start, "row_start", device), page_table.shape[1], n, rows,
            n * rows)
        self._made = (n * rows, ctypes.byref(self.sequences))

    def of(self, rows: int):
        """The batch for a call with so many rows in all (never changed after: another thread's call may be reading
        it)."""
        made = self._made
        if made[0] != rows:
            sequences = PagedSequences.from_buffer_copy(self.sequences)
            sequences.total_rows = rows
            made = self._made = (rows, ctypes.byref(sequences))
        return made[1]


def _paged_device(kv: PagedKv, batch: PagedBatch) -> int:
    if batch.device != kv.device:
        raise FoError(f"the page table is on GPU {batch.device}, the pool on GPU {kv.device}")
    return kv.device


def paged_append(kv: PagedKv, batch: PagedBatch, k, v, rope: Optional[Rope] = None, positions=None, q=None,
                 q_out=None, ctx=None):
    """fo_paged_append: rows k, v [rows][kv heads][head dim] into the batch's
    pages, keys rotated on the way when `rope` is given (at `positions`, else
    at their place in the cache; with a RopeAxes, fo_paged_append_by_axes, at
    `positions` [axes][rows]), and queries q rotated into q_out."""
    device = _paged_device(kv, batch)
    rk, rv = _rows(k, "k", device), _rows(v, "v", device)
    rows, _, dim = shape = k.shape
    if dim != kv.head_dim or v.shape != shape:
        raise FoError("paged_append: k and v must be [rows][kv heads][head dim] of the cache")
    rq = ro = None
    if q is not None:
        shape = q.shape
        if q_out is None or shape != q_out.shape or shape[0] != rows or shape[2] != dim:
            raise FoError("paged_append: q and q_out must be [rows][heads][head dim]")
        rq, ro = _rows(q, "q", device), _rows(q_out, "q_out", device)
    if rope is None and positions is not None:
        raise FoError("paged_append: positions are the rotation's, without rope there is nothing to do with them")
    ctx = _context(ctx, device)
    call = getattr(lib(), "fo_paged_append" if rope is None else rope.append_call)
    check(call(ctx.handle, kv.ref, batch.of(rows), rk, rv, rq, ro,
               None if rope is None else rope.at(positions, rows, device)))


def paged_attention(kv: PagedKv, batch: PagedBatch, q, out, sinks=None, scale=None, window=0, lse=None, ctx=None):
    """fo_paged_attention: q [rows][heads][head dim] over the batch's cached
    positions into `out`; scale None: 1 / sqrt(head dim)."""
    device = _paged_device(kv, batch)
    rq, ro = _rows(q, "q", device), _rows(out, "out", device)
    rows, heads, dim = shape = q.shape
    if dim != kv.head_dim or out.shape != shape:
        raise FoError("paged_attention: q and out must be [rows][heads][head dim] of the cache's width")
    ctx = _context(ctx, device)
    check(lib().fo_paged_attention(ctx.handle, kv.ref, batch.of(rows), rq,
                                   None if sinks is None else _floats(sinks, heads, "sinks", device),
                                   kv.scale if scale is None else scale, window, ro,
                                   None if lse is None else _floats(lse, rows * heads, "lse", device)))
    return out


def paged_window_attention(kv: PagedKv, batch: PagedBatch, q, out, window=0, first=0, sinks=None, scale=None,
                           lse=None, ctx=None):
    """fo_paged_window_attention: as paged_attention, for any number of rows
    (a prompt's too), over the newest `window` positions (0: all) and the
    `first` ones, which stay in sight behind them."""
    device = _paged_device(kv, batch)
    rq, ro = _rows(q, "q", device), _rows(out, "out", device)
    rows, heads, dim = shape = q.shape
    if dim != kv.head_dim or out.shape != shape:
        raise FoError("paged_window_attention: q and out must be [rows][heads][head dim] of the cache's width")
    ctx = _context(ctx, device)
    check(lib().fo_paged_window_attention(ctx.handle, kv.ref, batch.of(rows), rq,
                                          None if sinks is None else _floats(sinks, heads, "sinks", device),
                                          kv.scale if scale is None else scale, window, first, ro,
                                          None if lse is None else _floats(lse, rows * heads, "lse", device)))
    return out


class PagedGroups:
    """Groups of a batch's sequences that share their beginnings
    (fo_paged_groups): seq_start [groups + 1] and lens [groups] int32.  Group
    g's sequences seq_start[g] .. seq_start[g + 1] - 1 have their positions
    below lens[g] in the pages of the first of them.  The tensors are the
    caller's and may change between calls."""

    def __init__(self, seq_start, lens):
        if seq_start.numel() != lens.numel() + 1:
            raise FoError("seq_start must have one entry more than there are groups")
        self.keep, self.device = (seq_start, lens), lens.get_device()
        self.groups = PagedPrefixes(_device_ints(seq_start, "seq_start", self.device),
                                    _device_ints(lens, "lens", self.device), lens.numel())
        self.ref = ctypes.byref(self.groups)


def paged_prefix_attention(kv: PagedKv, batch: PagedBatch, groups: PagedGroups, q, out, sinks=None, scale=None,
                           lse=None, ctx=None):
    """fo_paged_prefix_attention: paged_attention of sequences whose groups
    share their beginnings, which are read once for a group."""
    device = _paged_device(kv, batch)
    if groups.device != device:
        raise FoError(f"the groups are on GPU {groups.device}, the call on GPU {device}")
    rq, ro = _rows(q, "q", device), _rows(out, "out", device)
    rows, heads, dim = shape = q.shape
    if dim != kv.head_dim or out.shape != shape:
        raise FoError("paged_prefix_attention: q and out must be [rows][heads][head dim] of the cache's width")
    ctx = _context(ctx, device)
    check(lib().fo_paged_prefix_attention(ctx.handle, kv.ref, batch.of(rows), groups.ref, rq,
                                          None if sinks is None else _floats(sinks, heads, "sinks", device),
                                          kv.scale if scale is None else scale, ro,
                                          None if lse is None else _floats(lse, rows * heads, "lse", device)))
    return out


class _DeviceArray:
    """A raw device pointer as a CUDA array (__cuda_array_interface__)."""

    def __init__(self, ptr, n, dtype):
        self.__cuda_array_interface__ = {"shape": (n,), "typestr": np.dtype(dtype).str, "data": (ptr, False),
                                         "version": 3, "strides": None}


def device_to_host(ptr, n, dtype):
    """n elements of device memory at `ptr` (e.g. from SplitPrefix.records)
    copied to a numpy array through torch (tests and tooling)."""
    import torch
    torch.cuda.synchronize()
    return torch.as_tensor(_DeviceArray(ptr, n, dtype), device="cuda").cpu().numpy().copy()
