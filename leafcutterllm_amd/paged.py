"""The paged K/V cache and its attention over the C ABI (lcmoe_kv_*).

Operands are device addresses (int, or None for NULL), as in
MoeFfn.forward_dev: of hip.DeviceBuffer.ptr, or of any other library's
device tensors.  Every call is enqueued on `stream` and returns at once.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from ._lib import check, lib


class KvDesc(C.Structure):
    """lcmoe_kv_desc (include/lcmoe.h)."""

    _fields_ = [
        ("n_head", C.c_int32), ("n_kv_head", C.c_int32), ("head_dim", C.c_int32),
        ("page_tokens", C.c_int32), ("n_pages", C.c_int32), ("max_pages", C.c_int32),
        ("kv_type", C.c_int32), ("act_type", C.c_int32), ("rope_positions", C.c_int32),
    ]


class KvPool(C.Structure):
    """lcmoe_kv_pool: device addresses of the pages and their scales."""

    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("scale", C.c_void_p)]


class KvBatch(C.Structure):
    """lcmoe_kv_batch: a ragged batch; starts, lens and pages are device
    addresses of int32 arrays."""

    _fields_ = [
        ("n_seq", C.c_int32), ("n_rows", C.c_int32), ("max_new", C.c_int32),
        ("starts", C.c_void_p), ("lens", C.c_void_p), ("pages", C.c_void_p),
    ]


_vp, _i64, _D, _P, _B = C.c_void_p, C.c_int64, C.POINTER(KvDesc), C.POINTER(KvPool), C.POINTER(KvBatch)
_SIGS = {
    "lcmoe_kv_sizes": [_D, C.POINTER(C.c_size_t), C.POINTER(C.c_size_t)],
    "lcmoe_rope_table": [C.c_float, C.c_int32, C.c_int32, _vp],
    "lcmoe_kv_append_dev": [_D, _P, _B, _vp, _i64, _vp, _i64, _vp, _vp],
    "lcmoe_kv_read_dev": [_D, _P, _B, _vp, _i64, _vp, _i64, _vp],
    "lcmoe_kv_attention_workspace": [_D, _B, C.POINTER(C.c_size_t)],
    "lcmoe_kv_attention_dev": [_D, _P, _B, _vp, _i64, _vp, C.c_float, _vp, _i64, _vp, C.c_size_t,
                               _vp],
}
_bound_lib = None


def _bound():
    global _bound_lib
    if _bound_lib is None:
        L = lib()
        for name, args in _SIGS.items():
            fn = getattr(L, name)
            fn.restype, fn.argtypes = C.c_int32, args
        _bound_lib = L
    return _bound_lib


def kv_sizes(desc: KvDesc):
    """(bytes of the pool's k and of its v, bytes of its scales)."""
    n, s = C.c_size_t(), C.c_size_t()
    check(_bound().lcmoe_kv_sizes(C.byref(desc), C.byref(n), C.byref(s)), "lcmoe_kv_sizes")
    return n.value, s.value


def rope_table(theta: float, head_dim: int, n_pos: int) -> np.ndarray:
    """[n_pos, head_dim / 2, 2]: cosine and sine of each position's angles."""
    out = np.empty((max(n_pos, 0), max(head_dim, 0) // 2, 2), np.float32)
    check(_bound().lcmoe_rope_table(theta, head_dim, n_pos, out.ctypes.data), "lcmoe_rope_table")
    return out


def kv_append_dev(desc: KvDesc, pool: KvPool, batch: KvBatch, k: int, ld_k: int, v: int, ld_v: int,
                  rope: int | None = None, stream: int | None = None) -> None:
    """Appends the batch's keys (rotated with `rope`) and values to the cache."""
    check(_bound().lcmoe_kv_append_dev(desc, pool, batch, k, ld_k, v, ld_v, rope, stream),
          "lcmoe_kv_append_dev")


def kv_read_dev(desc: KvDesc, pool: KvPool, batch: KvBatch, k: int, ld_k: int, v: int, ld_v: int,
                stream: int | None = None) -> None:
    """The cached values at the batch's positions, as rows of k and v."""
    check(_bound().lcmoe_kv_read_dev(desc, pool, batch, k, ld_k, v, ld_v, stream),
          "lcmoe_kv_read_dev")


def kv_attention_workspace(desc: KvDesc, batch: KvBatch) -> int:
    """Bytes that kv_attention_dev needs for this desc and batch size."""
    n = C.c_size_t()
    check(_bound().lcmoe_kv_attention_workspace(C.byref(desc), C.byref(batch), C.byref(n)),
          "lcmoe_kv_attention_workspace")
    return n.value


def kv_attention_dev(desc: KvDesc, pool: KvPool, batch: KvBatch, q: int, ld_q: int,
                     rope: int | None, scale: float, out: int, ld_out: int,
                     workspace: int | None, workspace_bytes: int,
                     stream: int | None = None) -> None:
    """Causal attention of the batch's rows over the cache, q rotated with `rope`."""
    check(_bound().lcmoe_kv_attention_dev(desc, pool, batch, q, ld_q, rope, scale, out, ld_out,
                                          workspace, workspace_bytes, stream),
          "lcmoe_kv_attention_dev")


__all__ = ["KvDesc", "KvPool", "KvBatch", "kv_sizes", "rope_table", "kv_append_dev", "kv_read_dev",
           "kv_attention_workspace", "kv_attention_dev"]
