"""Log probabilities, entropy and top alternatives on the GPU against float64."""
import numpy as np
import pytest

import leafcutterllm_amd as L
from kv_ref import ACTS, from_bits, to_bits
from leafcutterllm_amd import hip

pytestmark = pytest.mark.gpu


def reference(x, given, n_top):
    """The definition in float64; x [rows, vocab]."""
    rows, V = x.shape
    with np.errstate(all="ignore"):
        m = x.max(1, keepdims=True)
        p = np.where(x == -np.inf, 0, np.exp(x - m))
        z = p.sum(1, keepdims=True)
        lp = x - m - np.log(z)
        ent = -(np.where(p > 0, p * lp, 0)).sum(1) / z[:, 0]
    empty = np.all(x == -np.inf, 1)
    lp[empty], ent[empty] = -np.inf, 0
    bad = np.isnan(x).any(1) | (x == np.inf).any(1)
    lp[bad], ent[bad] = np.nan, np.nan
    ok = (given >= 0) & (given < V)
    glp = np.where(ok, np.take_along_axis(lp, np.where(ok, given, 0), 1), 0)
    key = np.where(np.isnan(x), -np.inf, x)
    ids = np.argsort(-key, axis=1, kind="stable")[:, :n_top]
    return glp, ent, ids, np.take_along_axis(lp, ids, 1)


def run(x, given, n_top, act, ld=None, offset=0, entropy=True):
    """x [rows, vocab] as the activation type's array."""
    rows, V = x.shape
    ld = ld or V
    flat = np.zeros(offset + rows * ld, x.dtype)
    flat[offset:].reshape(rows, ld)[:, :V] = x
    xb = hip.DeviceBuffer(flat.nbytes).upload(flat)
    ng = given.shape[1]
    gb = hip.DeviceBuffer(max(4 * rows * ng, 4))
    if ng:
        gb.upload(np.ascontiguousarray(given, np.int32))
    outs = [np.full((rows, ng), 7, np.float32), np.full(rows, 7, np.float32),
            np.full((rows, n_top), 7, np.int32), np.full((rows, n_top), 7, np.float32)]
    bufs = [hip.DeviceBuffer(max(o.nbytes, 4)) for o in outs]
    for o, b in zip(outs, bufs):
        if o.size:
            b.upload(o)
    n = L.logprobs_workspace(ACTS[act], rows, V, ng, n_top)
    ws = hip.DeviceBuffer(max(n, 16)).upload(np.full(max(n, 16), 0xFF, np.uint8))
    st = hip.Stream()
    L.logprobs_dev(ACTS[act], xb.ptr + offset * x.itemsize, ld, rows, V, gb.ptr, ng, bufs[0].ptr,
                   bufs[1].ptr if entropy else None, n_top, bufs[2].ptr, bufs[3].ptr, ws.ptr, n,
                   st.ptr)
    st.synchronize()
    return [b.download(o) if o.size else o for o, b in zip(outs, bufs)]


def check(x, given, n_top, act, **kw):
    got = run(x, given, n_top, act, **kw)
    v = from_bits(x, act)
    want = reference(v, given, n_top)
    k = min(n_top, v.shape[1])
    np.testing.assert_array_equal(got[2][:, :k], want[2])
    assert (got[2][:, k:] == -1).all() and (got[3][:, k:] == -np.inf).all()
    fin = np.where(np.isfinite(v), np.abs(v), 0).max(1, keepdims=True)
    # Z: exponentials of arguments off by 2^-23 of their size, to 1 ulp, summed
    # in f32 chains of at most 200 steps of one sign; log p: three f32 values
    # of at most 2 max|x| + log V added.  The entropy's sum has terms of one
    # sign and of the same kind.
    span = 2 * fin + np.log(v.shape[1])
    tol = (span * 2 + 220) * 2.0**-23
    for i in (0, 1, 3):
        g, w = got[i][:, :k] if i == 3 else got[i], want[i]
        t = tol if i != 1 else tol[:, 0] * (1 + np.log(v.shape[1]))
        np.testing.assert_array_equal(np.isnan(g), np.isnan(w))
        np.testing.assert_array_equal(g == -np.inf, w == -np.inf)
        with np.errstate(invalid="ignore"):
            d = np.abs(g - w)
        assert np.all((d <= t) | ~np.isfinite(w)), (i, np.nanmax(d), t.max())
    return got


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,V", [(1, 1), (3, 2), (2, 31), (5, 255), (4, 257), (2, 1000), (7, 4099),
                                    (1, 32000), (33, 32000), (3, 131075), (1, 600001), (1500, 300)])
def test_sizes(act, rows, V):
    rng = np.random.default_rng(rows + V)
    x = to_bits((rng.standard_normal((rows, V)) * 3).astype(np.float32), act)
    given = rng.integers(0, V, (rows, 2))
    for n_top, ng in ((0, 2), (1, 0), (20, 1), (32, 2)):
        check(x, given[:, :ng], n_top, act)


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("offset,pad", [(1, 1), (3, 6), (0, 5)])
def test_rows_apart_and_unaligned(act, offset, pad):
    rng = np.random.default_rng(offset + pad)
    for V in (61, 5003, 40000):
        x = to_bits((rng.standard_normal((3, V)) * 3).astype(np.float32), act)
        check(x, rng.integers(0, V, (3, 1)), 7, act, ld=V + pad, offset=offset)


@pytest.mark.parametrize("V", [40, 3000, 70000])
def test_ties_take_the_lowest_id(V):
    rng = np.random.default_rng(V)
    x = np.stack([np.zeros(V), np.where(rng.random(V) < 0.5, -0.0, 0.0), rng.integers(0, 3, V),
                  np.full(V, -5.0), np.arange(V) // (V // 8)]).astype(np.float32)
    check(x, np.zeros((5, 1), int), 32, "f32")


@pytest.mark.parametrize("V", [5000, 130000])
def test_the_largest_in_a_thread(V):
    """Sorted rows, and all of the largest at one stride: elements of a single
    thread, or of neighbours."""
    x = np.zeros((5, V), np.float32)
    x[0], x[1] = np.arange(V) / V, -np.arange(V) / V
    for r, stride in ((2, 256), (3, 1024), (4, 8)):
        at = np.arange(3, V, stride)[:64]
        x[r, at] = 5 + np.arange(len(at)) / 64
    check(x, np.zeros((5, 1), int), 32, "f32")


@pytest.mark.parametrize("act,V", [("f32", 8192), ("f32", 32768), ("f32", 100003), ("f16", 32768)])
def test_large_ones_side_by_side(act, V):
    """4 of every 64 groups of 16 bytes hold all of the largest, so that a
    bound from the largest element of each group's lane lies below them all."""
    rng = np.random.default_rng(V)
    g = 4 if act == "f32" else 8
    x = rng.random((3, V))
    x[(slice(None), np.arange(V) // g % 64 < 4)] += 5
    check(to_bits(x.astype(np.float32), act), np.zeros((3, 1), int), 32, act)


@pytest.mark.parametrize("span", [8192, 32768])
def test_large_ones_in_every_part(span):
    """31 of the largest in each of 40 parts of a row, and 40 in one."""
    rng = np.random.default_rng(span)
    x = rng.random((40, span)).astype(np.float32)
    for r in range(40):
        x[r, rng.choice(span, 40 if r == 17 else 31, replace=False)] += 5
    check(x.reshape(1, -1), np.zeros((1, 1), int), 32, "f32")


@pytest.mark.parametrize("V", [100, 5000, 200000])
def test_masked_and_nonfinite(V):
    rng = np.random.default_rng(V)
    x = (rng.standard_normal((9, V)) * 3).astype(np.float32)
    x[0] = -np.inf                       # nothing left
    x[1, 5:] = -np.inf                   # five tokens left
    x[2, : V - 1] = -np.inf              # one token left, the last
    x[3] = np.finfo(np.float32).min      # the type's lowest value everywhere
    x[4, 1:] = np.finfo(np.float32).min
    x[5, V // 2] = np.nan
    x[6, 7] = np.inf
    x[7] = -np.inf
    x[7, V // 3] = np.nan                # NaN among nothing
    x[8] += 1e4                          # far from zero
    got = check(x, np.tile([0, V - 1], (9, 1)), 10, "f32")
    assert got[1][0] == 0 and got[1][2] == 0 and np.isnan(got[1][[5, 6, 7]]).all()


def test_ids_outside_the_vocabulary():
    x = np.zeros((2, 300), np.float32)
    given = np.array([[-1, 0, 300, 299], [2**31 - 1, -2**31, -100, 5]])
    got = check(x, given, 0, "f32")
    assert (got[0] == np.where((given >= 0) & (given < 300), got[0], 0)).all()


def test_results_not_wanted():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((4, 900)).astype(np.float32)
    got = run(x, np.zeros((4, 0), np.int32), 3, "f32", entropy=False)
    assert (got[1] == 7).all()
    np.testing.assert_array_equal(got[2], reference(x.astype(np.float64), np.zeros((4, 0), int), 3)[2])


def test_rows_past_the_grid():
    rng = np.random.default_rng(2)
    x = rng.standard_normal((70000, 40)).astype(np.float32)
    check(x, rng.integers(0, 40, (70000, 1)), 2, "f32")


def test_host_form_and_repeats():
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((20, 50000)) * 4).astype(np.float32)
    given = rng.integers(0, 50000, (20, 3))
    first = L.logprobs(x, given, 12)
    for a, b in zip(first, run(x, given, 12, "f32")):
        np.testing.assert_array_equal(a, b)
    for _ in range(3):
        for a, b in zip(first, L.logprobs(x, given, 12)):
            np.testing.assert_array_equal(a, b)
    h = x.astype(np.float16)
    np.testing.assert_array_equal(L.logprobs(h, given, 5)[2], run(h, given, 5, "f16")[2])
