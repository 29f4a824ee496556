"""Log probabilities of rows of logits over the C ABI (lcmoe_logprobs*)."""
from __future__ import annotations

import ctypes as C

import numpy as np

from ._lib import TYPE_F16, TYPE_F32, LcmoeError, check, lib

_vp, _i32, _i64 = C.c_void_p, C.c_int32, C.c_int64
_SIGS = {
    "lcmoe_logprobs_workspace": [_i32, _i32, _i32, _i32, _i32, C.POINTER(C.c_size_t)],
    "lcmoe_logprobs_dev": [_i32, _vp, _i64, _i32, _i32, _vp, _i32, _vp, _vp, _i32, _vp, _vp, _vp,
                           C.c_size_t, _vp],
    "lcmoe_logprobs": [_i32, _vp, _i64, _i32, _i32, _vp, _i32, _vp, _vp, _i32, _vp, _vp],
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


def logprobs_workspace(type: int, n_rows: int, vocab: int, n_given: int, n_top: int) -> int:
    """Bytes that logprobs_dev needs for these sizes."""
    n = C.c_size_t()
    check(_bound().lcmoe_logprobs_workspace(type, n_rows, vocab, n_given, n_top, C.byref(n)),
          "lcmoe_logprobs_workspace")
    return n.value


def logprobs_dev(type: int, logits: int, ld: int, n_rows: int, vocab: int, given: int | None,
                 n_given: int, given_lp: int | None, entropy: int | None, n_top: int,
                 top_id: int | None, top_lp: int | None, workspace: int | None,
                 workspace_bytes: int, stream: int | None = None) -> None:
    """lcmoe_logprobs_dev: device addresses, enqueued on `stream`."""
    check(_bound().lcmoe_logprobs_dev(type, logits, ld, n_rows, vocab, given, n_given, given_lp,
                                      entropy, n_top, top_id, top_lp, workspace, workspace_bytes,
                                      stream), "lcmoe_logprobs_dev")


def logprobs(logits: np.ndarray, given=None, n_top: int = 0):
    """(log probabilities of `given` [rows, n], entropy [rows], ids and log
    probabilities of the n_top largest logits [rows, n_top]) of f32 or f16
    logits [rows, vocab]: lcmoe_logprobs on the GPU."""
    x = np.atleast_2d(logits)
    if x.ndim != 2 or x.dtype not in (np.float32, np.float16):
        raise LcmoeError(1, "logprobs", "logits must be f32 or f16, [rows, vocab]")
    x = np.ascontiguousarray(x)
    rows, vocab = x.shape
    g = np.empty((rows, 0), np.int32) if given is None else np.asarray(given, np.int32)
    if g.ndim == 1:
        g = g[:, None]
    if g.ndim != 2 or g.shape[0] != rows:
        raise LcmoeError(1, "logprobs", f"given must be [{rows}, n]")
    if n_top < 0:
        raise LcmoeError(1, "logprobs", f"n_top={n_top}")
    g = np.ascontiguousarray(g)
    lp, ent = np.empty(g.shape, np.float32), np.empty(rows, np.float32)
    ids, top = np.empty((rows, n_top), np.int32), np.empty((rows, n_top), np.float32)
    check(_bound().lcmoe_logprobs(TYPE_F32 if x.dtype == np.float32 else TYPE_F16, x.ctypes.data,
                                  vocab, rows, vocab, g.ctypes.data, g.shape[1], lp.ctypes.data,
                                  ent.ctypes.data, n_top, ids.ctypes.data, top.ctypes.data),
          "lcmoe_logprobs")
    return lp, ent, ids, top


__all__ = ["logprobs", "logprobs_dev", "logprobs_workspace"]
