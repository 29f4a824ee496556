"""A paged K/V cache, its attention and log probabilities in float64 numpy:
the definitions that include/lcmoe.h writes down, without the library's
layout.  Test infrastructure only."""
from __future__ import annotations

import ctypes as C

import numpy as np

import leafcutterllm_amd as L
from leafcutterllm_amd import hip

ACTS = {"f32": L.TYPE_F32, "f16": L.TYPE_F16, "bf16": L.TYPE_BF16}
KVS = {"f16": L.TYPE_F16, "i8": L.TYPE_I8}
# a rounding's largest error, relative to the value
HALF_STEP = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}


def to_bits(x, act):
    """f32 values as the activation type's array (bf16 as its upper 16 bits, to
    nearest even)."""
    x = np.ascontiguousarray(x, np.float32)
    if act == "f32":
        return x
    if act == "f16":
        return x.astype(np.float16)
    u = x.view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bits(a, act):
    """The activation type's array as float64."""
    if act == "bf16":
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


def rotate(x, cs):
    """x [..., hd] by (cos, sin) = cs [..., hd / 2, 2]."""
    h = x.shape[-1] // 2
    c, s = cs[..., 0].astype(np.float64), cs[..., 1].astype(np.float64)
    lo, hi = x[..., :h], x[..., h:]
    return np.concatenate([lo * c - hi * s, lo * s + hi * c], -1)


class RefCache:
    """One layer's pages.  I8: codes and a scale per page, head and keys /
    values; F16: the rounded values."""

    def __init__(self, n_pages, KVH, hd, page, kv):
        self.page, self.kv = page, kv
        self.data = np.zeros((2, n_pages, KVH, page, hd))
        self.scale = np.zeros((2, n_pages, KVH), np.float32)

    def append(self, pages, len0, k, v):
        """k (rotated), v [T, KVH, hd] float64 at positions len0 on."""
        for j, x in enumerate((k, v)):
            t = 0
            while t < x.shape[0]:
                p, slot = divmod(len0 + t, self.page)
                n = min(self.page - slot, x.shape[0] - t)
                if p >= len(pages):
                    break
                if 0 <= pages[p] < self.data.shape[1]:
                    self._into(j, pages[p], slot, x[t:t + n].transpose(1, 0, 2))
                t += n

    def _into(self, j, page, slot, x):
        if self.kv == "f16":
            with np.errstate(over="ignore"):
                self.data[j, page, :, slot:slot + x.shape[1]] = x.astype(np.float16)
            return
        old = self.scale[j, page] if slot else np.zeros(x.shape[0], np.float32)
        most = np.where(np.isfinite(x), np.abs(x), 0).max((1, 2))
        new = np.maximum(old, (most / 127).astype(np.float32))
        d, s = self.data[j, page], new.astype(np.float64)
        with np.errstate(divide="ignore", invalid="ignore"):
            ratio = np.where(new > old, old.astype(np.float64) / s, 1.0)
            d[:, :slot] = np.rint(d[:, :slot] * ratio[:, None, None])
            q = np.rint(x / s[:, None, None])
        d[:, slot:slot + x.shape[1]] = np.where(np.isnan(q), 0, np.clip(q, -127, 127))
        self.scale[j, page] = new

    def values(self, j, pages, n):
        """[n, KVH, hd] as held, and which positions are there."""
        pages = np.asarray(pages)[: -(-n // self.page)]
        there = (pages >= 0) & (pages < self.data.shape[1])
        x = self.data[j, np.where(there, pages, 0)]
        if self.kv == "i8":
            # a value is the f32 product of its code and its scale
            x = (x.astype(np.float32) * self.scale[j, np.where(there, pages, 0)][..., None, None]).astype(np.float64)
        x = x.transpose(0, 2, 1, 3).reshape(-1, *x.shape[1:2], x.shape[3])[:n]
        return x, np.repeat(there, self.page)[:n]


def attend(q, k, v, pos, there, scale):
    """q [H, hd] at position pos over k, v [n, KVH, hd]: out [H, hd], and what
    its error is counted in: the largest p and the keys seen, the sum of p |v|,
    the largest scores of |q| |k| and of max |q| |k|."""
    H, G = q.shape[0], q.shape[0] // k.shape[1]
    see = there & (np.arange(k.shape[0]) <= pos)
    out, size = np.zeros_like(q), np.zeros_like(q)
    top, mag, most = np.zeros((H, 1)), np.zeros((H, 1)), np.zeros((H, 1))
    for h in range(H if see.any() else 0):
        kk, vv = k[see, h // G], v[see, h // G]
        with np.errstate(invalid="ignore", over="ignore"):
            s = scale * (kk @ q[h])
            p = np.exp(s - s.max())
            p /= p.sum()
            out[h], size[h], top[h] = p @ vv, p @ np.abs(vv), p.max()
            mag[h] = scale * (np.abs(kk) @ np.abs(q[h])).max()
            most[h] = scale * (np.abs(kk).sum(1) * np.abs(q[h]).max()).max()
    return out, size, top, mag, most, see.sum()


class Graph:
    """What `work` enqueues on the stream, captured once; replay() runs it."""

    def __init__(self, stream, work):
        rt, self.stream = hip.rt(), stream
        for name, args in (("hipStreamBeginCapture", [C.c_void_p, C.c_int]),
                           ("hipStreamEndCapture", [C.c_void_p, C.POINTER(C.c_void_p)]),
                           ("hipGraphInstantiate", [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p,
                                                    C.c_void_p, C.c_size_t]),
                           ("hipGraphLaunch", [C.c_void_p, C.c_void_p]),
                           ("hipGraphDestroy", [C.c_void_p]), ("hipGraphExecDestroy", [C.c_void_p])):
            getattr(rt, name).argtypes = args
        g, self.exec = C.c_void_p(), C.c_void_p()
        assert rt.hipStreamBeginCapture(stream.ptr, 2) == 0  # relaxed
        work()
        assert rt.hipStreamEndCapture(stream.ptr, C.byref(g)) == 0
        assert rt.hipGraphInstantiate(C.byref(self.exec), g, None, None, 0) == 0
        assert rt.hipGraphDestroy(g) == 0

    def replay(self):
        assert hip.rt().hipGraphLaunch(self.exec, self.stream.ptr) == 0

    def close(self):
        assert hip.rt().hipGraphExecDestroy(self.exec) == 0


class Rig:
    """A pool on the GPU and its RefCache, driven together."""

    def __init__(self, H, KVH, hd, page, kv, act, n_pages, max_pages, absolute=True, theta=10000.0,
                 rope=True):
        self.H, self.KVH, self.hd, self.page, self.kv, self.act = H, KVH, hd, page, kv, act
        self.absolute, self.n_pages, self.max_pages = absolute, n_pages, max_pages
        self.desc = L.KvDesc(H, KVH, hd, page, n_pages, max_pages, KVS[kv], ACTS[act],
                             L.ROPE_ABSOLUTE if absolute else L.ROPE_PER_CALL)
        n, ns = L.kv_sizes(self.desc)
        # every byte 0x7e: NaN as f16, 126 as a code, 8.5e37 as a scale
        self.bufs = [hip.DeviceBuffer(n).upload(np.full(n, 0x7E, np.uint8)) for _ in range(2)]
        self.bufs.append(hip.DeviceBuffer(max(ns, 8)).upload(np.full(max(ns, 8), 0x7E, np.uint8)))
        self.pool = L.KvPool(self.bufs[0].ptr, self.bufs[1].ptr, self.bufs[2].ptr if ns else None)
        self.ref = RefCache(n_pages, KVH, hd, page, kv)
        self.table = L.rope_table(theta, hd, max_pages * page) if rope else None
        self.rope = hip.DeviceBuffer(self.table.nbytes).upload(self.table) if rope else None
        self.stream = hip.Stream()

    def batch(self, lens, new, pages, max_new=None, starts=True, n_rows=None):
        """(KvBatch, the buffers that it points to)."""
        at = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        keep = [hip.DeviceBuffer(4 * len(at)).upload(at),
                hip.DeviceBuffer(max(4 * len(lens), 4)).upload(np.asarray(lens, np.int32)),
                hip.DeviceBuffer(max(4 * len(lens) * self.max_pages, 4)).upload(
                    np.ascontiguousarray(pages, np.int32))]
        return L.KvBatch(len(lens), int(at[-1]) if n_rows is None else n_rows,
                         max(new, default=0) if max_new is None else max_new,
                         keep[0].ptr if starts else None, keep[1].ptr, keep[2].ptr), keep

    def _positions(self, lens, new):
        return [(b, i, lens[b] + i) for b in range(len(lens)) for i in range(new[b])]

    def _rotated(self, x, lens, new):
        if self.table is None:
            return x
        rot = [p if self.absolute else i for _, i, p in self._positions(lens, new)]
        return rotate(x, self.table[np.minimum(rot, len(self.table) - 1)][:, None])

    def append(self, lens, new, pages, k, v, batch=None):
        """k, v [N, KVH, hd] f32: into the GPU's pool, from one buffer whose
        rows hold the keys, the values and a tail, and into the reference."""
        N, row = k.shape[0], self.KVH * self.hd
        x = np.concatenate([k.reshape(N, row), v.reshape(N, row), np.zeros((N, 8), np.float32)], 1)
        bits = to_bits(x, self.act)
        buf = hip.DeviceBuffer(bits.nbytes).upload(bits)
        b, keep = batch or self.batch(lens, new, pages)
        L.kv_append_dev(self.desc, self.pool, b, buf.ptr, 2 * row + 8, buf.ptr + row * bits.itemsize,
                        2 * row + 8, self.rope and self.rope.ptr, self.stream.ptr)
        self.stream.synchronize()
        y = from_bits(bits, self.act)
        kr = self._rotated(y[:, :row].reshape(N, self.KVH, self.hd), lens, new)
        vr = y[:, row:2 * row].reshape(N, self.KVH, self.hd)
        at = 0
        for s in range(len(lens)):
            self.ref.append(pages[s], lens[s], kr[at:at + new[s]], vr[at:at + new[s]])
            at += new[s]

    def read(self, lens, new, pages):
        """The GPU's cache at those positions, as the activation type holds it."""
        N, row = sum(new), self.KVH * self.hd
        out = [hip.DeviceBuffer(N * row * (4 if self.act == "f32" else 2)) for _ in range(2)]
        b, keep = self.batch(lens, new, pages)
        L.kv_read_dev(self.desc, self.pool, b, out[0].ptr, row, out[1].ptr, row, self.stream.ptr)
        self.stream.synchronize()
        dt = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}[self.act]
        return [from_bits(o.download(np.empty((N, self.KVH, self.hd), dt)), self.act) for o in out]

    def check_held(self, lens, pages):
        """Every value that the sequences hold against the reference."""
        got = self.read([0] * len(lens), list(lens), pages)
        for j in range(2):
            want = np.concatenate([self.ref.values(j, pages[b], n)[0] * self.ref.values(j, pages[b], n)[1][:, None, None]
                                   for b, n in enumerate(lens)])
            if self.kv == "i8" or self.act != "f32":
                # codes and scales are the reference's; the result is rounded once more
                bits = to_bits(want.astype(np.float32), self.act)
                np.testing.assert_array_equal(got[j], from_bits(bits, self.act))
            else:
                np.testing.assert_array_equal(got[j], want)

    def attention(self, lens, new, pages, q, scale=None, batch=None, extra_rows=0, offset=0):
        """out [N + extra_rows, H, hd] float64 of q [N, H, hd] f32."""
        N, row = q.shape[0], self.H * self.hd
        scale = self.hd ** -0.5 if scale is None else scale
        bits = to_bits(q.reshape(N, row), self.act)
        it = bits.itemsize
        ld = row + (8 if offset == 0 else 3)
        rows = np.zeros((N, ld), bits.dtype)
        rows[:, :row] = bits
        qb = hip.DeviceBuffer(rows.nbytes + offset * it)
        flat = np.concatenate([np.zeros(offset, bits.dtype), rows.reshape(-1)])
        qb.upload(flat)
        out = np.full((N + extra_rows, ld), 7, bits.dtype)
        ob = hip.DeviceBuffer(out.nbytes + offset * it)
        ob.upload(np.concatenate([np.full(offset, 7, bits.dtype), out.reshape(-1)]))
        b, keep = batch or self.batch(lens, new, pages, n_rows=N + extra_rows)
        n = L.kv_attention_workspace(self.desc, b)
        ws = hip.DeviceBuffer(max(n, 16)).upload(np.full(max(n, 16), 0xFF, np.uint8))
        L.kv_attention_dev(self.desc, self.pool, b, qb.ptr + offset * it, ld,
                           self.rope and self.rope.ptr, scale, ob.ptr + offset * it, ld, ws.ptr, n,
                           self.stream.ptr)
        self.stream.synchronize()
        flat = ob.download(np.empty(offset + out.size, bits.dtype))
        got = flat[offset:].reshape(out.shape)
        assert (flat[:offset] == 7).all() and (got[:, row:] == 7).all() and (got[N:] == 7).all()
        return from_bits(got[:N, :row], self.act).reshape(N, self.H, self.hd)

    def check_attention(self, lens, new, pages, q, scale=None, got=None, every=1, **kw):
        """Against float64, to a bound that counts the kernel's roundings; of
        each sequence's rows the last and `every` so many."""
        got = self.attention(lens, new, pages, q, scale, **kw) if got is None else got
        scale = self.hd ** -0.5 if scale is None else scale
        qs = self._rotated(from_bits(to_bits(q, self.act), self.act), lens, new)
        at = 0
        for b in range(len(lens)):
            n = lens[b] + new[b]
            if not new[b]:
                continue
            k, there = self.ref.values(0, pages[b], n)
            v, _ = self.ref.values(1, pages[b], n)
            for i in range(new[b]):
                if (new[b] - 1 - i) % every:
                    at += 1
                    continue
                want, size, *by = attend(qs[at], k, v, lens[b] + i, there, scale)
                vmax = np.abs(v[there]).max(initial=0.0)
                tol = self.bound(size, *by, vmax) + HALF_STEP[self.act] * (np.abs(want) + size * 2.0**-9)
                assert np.all(np.isfinite(got[at])), (b, i)
                worst = np.abs(got[at] - want) - tol
                assert worst.max() <= 0, (b, i, np.abs(got[at] - want).max(), tol.max())
                at += 1
        return got

    def bound(self, size, top, mag, most, n, vmax):
        """How far an output may be off before its last rounding.

        q is rotated in f32 (2^-23 of its pair) and enters as three 8-bit or two
        f16 pieces where activations are f32, else as two 8-bit pieces or one
        f16: to 2^-21 or 2^-10 of itself, and in 8-bit pieces to 2^-24 or 2^-16
        of the row's largest.  The score is an f32 sum of at most head_dim + 16
        steps.  A score off by e multiplies its p by e^e and the others' share
        by as much: e^(2 e).  p enters as q does, in 8-bit pieces to 2^-23 or
        2^-15 of the row's largest (p times its page's scale over the largest
        of 64 tokens, at most 1), for each of n keys.  The sums of p and of p v
        are f32 chains of at most 64 + n / 64 steps."""
        fine = self.act == "f32"
        rel, part = (2.0**-21, 2.0**-24) if fine else (2.0**-10, 2.0**-16)
        e = mag * (rel + 2.0**-22 + (self.hd + 16) * 2.0**-24) + most * part + 2.0**-22
        chain = (64 + n / 64) * 2.0**-23
        parts = n * top * vmax * 2 * part if self.kv == "i8" else 0.0
        return size * (np.expm1(2 * e) + 2 * rel + chain) + parts
