"""The paged K/V cache on the GPU against float64: append, read back and
attention, on pools that start out as NaN."""
import numpy as np
import pytest

import leafcutterllm_amd as L
from kv_ref import ACTS, Graph, Rig, from_bits, to_bits
from leafcutterllm_amd import hip

pytestmark = pytest.mark.gpu


def normal(rng, *shape, scale=1.0):
    return (rng.standard_normal(shape) * scale).astype(np.float32)


def tables(rng, n_pages, max_pages, held):
    """A page table whose sequences hold `held` pages each, in any order."""
    order = rng.permutation(n_pages)
    t = np.full((len(held), max_pages), -1, np.int32)
    at = 0
    for b, n in enumerate(held):
        t[b, :n] = order[at:at + n]
        at += n
    return t


def fill(rig, rng, lens, pages, scale=1.0):
    """Appends lens[b] tokens to each sequence in one call."""
    N = sum(lens)
    rig.append([0] * len(lens), list(lens), pages, normal(rng, N, rig.KVH, rig.hd, scale=scale),
               normal(rng, N, rig.KVH, rig.hd, scale=scale))


# head sizes whose units end in 32 dims or in padded ones, every page size
@pytest.mark.parametrize("kv", ["i8", "f16"])
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd,KVH,page", [(16, 3, 16), (32, 2, 64), (64, 1, 16), (80, 2, 32),
                                         (96, 2, 16), (128, 2, 128), (256, 1, 256)])
def test_append_and_read(kv, act, hd, KVH, page):
    rng = np.random.default_rng(hd + page)
    rig = Rig(KVH, KVH, hd, page, kv, act, 40, 8)
    steps = [[3, 0, page, 2 * page + 1], [1, 1, 1, 1], [page - 3, 5, 0, page], [1, 2, 20, 1]]
    pages = tables(rng, 40, 8, [8, 8, 8, 8])
    lens = [0, 0, 0, 0]
    for i, new in enumerate(steps):
        # later tokens are larger: pages whose scale grows, and others
        N, s = sum(new), [1.0, 2.0, 0.5, 3.0][i]
        rig.append(lens, new, pages, normal(rng, N, KVH, hd, scale=s), normal(rng, N, KVH, hd, scale=s))
        lens = [a + b for a, b in zip(lens, new)]
        rig.check_held(lens, pages)


@pytest.mark.parametrize("kv", ["i8", "f16"])
@pytest.mark.parametrize("absolute,rope", [(False, True), (True, False)])
def test_positions(kv, absolute, rope):
    """Rotation by the number in the call, and none."""
    rng = np.random.default_rng(3)
    rig = Rig(4, 2, 64, 16, kv, "f32", 20, 6, absolute=absolute, rope=rope)
    pages = tables(rng, 20, 6, [6, 6])
    fill(rig, rng, [17, 30], pages)
    new = [5, 2]
    rig.append([17, 30], new, pages, normal(rng, 7, 2, 64), normal(rng, 7, 2, 64))
    rig.check_held([22, 32], pages)
    rig.check_attention([17, 30], new, pages, normal(rng, 7, 4, 64))


@pytest.mark.parametrize("kv", ["i8", "f16"])
def test_one_token_at_a_time(kv):
    """A decode: the scale of a page grows as it fills, attention after each."""
    rng = np.random.default_rng(5)
    rig = Rig(6, 2, 64, 16, kv, "f32", 12, 4)
    pages = tables(rng, 12, 4, [4, 4, 4])
    lens = [0, 15, 31]
    fill(rig, rng, lens, pages)
    for i in range(20):
        rig.append(lens, [1, 1, 1], pages, normal(rng, 3, 2, 64, scale=1 + i / 4),
                   normal(rng, 3, 2, 64, scale=1 + i / 4))
        rig.check_attention(lens, [1, 1, 1], pages, normal(rng, 3, 6, 64))
        lens = [n + 1 for n in lens]
    rig.check_held(lens, pages)


@pytest.mark.parametrize("kv", ["i8", "f16"])
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd,H,KVH,page", [(16, 4, 4, 16), (32, 3, 1, 32), (64, 17, 1, 16),
                                           (80, 4, 2, 64), (96, 5, 5, 16), (128, 8, 2, 16),
                                           (160, 2, 1, 16), (192, 4, 1, 64), (224, 2, 2, 16),
                                           (256, 8, 1, 256)])
def test_attention_of_a_ragged_batch(kv, act, hd, H, KVH, page):
    """Nothing cached, nothing new, single tokens, a piece behind a history,
    and a prompt past the tile edges, in one call."""
    rng = np.random.default_rng(hd + H + page)
    lens = [0, 40, 200, 0, 63, 130, 1, 15]
    new = [1, 0, 1, 0, 17, 70, 33, 1]
    held = [-(-(a + b) // page) for a, b in zip(lens, new)]
    most = max(held) + 1
    rig = Rig(H, KVH, hd, page, kv, act, sum(held) + 2, most)
    pages = tables(rng, rig.n_pages, most, held)
    fill(rig, rng, lens, pages)
    N = sum(new)
    rig.append(lens, new, pages, normal(rng, N, KVH, hd), normal(rng, N, KVH, hd))
    rig.check_attention(lens, new, pages, normal(rng, N, H, hd), extra_rows=5)


# around the 64-token steps and the pages, for one token and for a few
@pytest.mark.parametrize("kv", ["i8", "f16"])
@pytest.mark.parametrize("new", [1, 2, 5, 16])
@pytest.mark.parametrize("n", [0, 1, 15, 16, 47, 63, 64, 65, 127, 128, 255, 257, 700])
def test_attention_lengths(kv, new, n):
    rng = np.random.default_rng(n + new)
    rig = Rig(4, 2, 64, 16, kv, "f32", 60, 50)
    pages = tables(rng, 60, 50, [-(-(n + new) // 16)])
    if n:
        fill(rig, rng, [n], pages)
    rig.append([n], [new], pages, normal(rng, new, 2, 64), normal(rng, new, 2, 64))
    q = normal(rng, new, 4, 64, scale=3.0)  # peaked rows among them
    got = rig.check_attention([n], [new], pages, q)
    b, keep = rig.batch([n], [new], pages, starts=False)
    np.testing.assert_array_equal(got, rig.attention([n], [new], pages, q, batch=(b, keep)))


@pytest.mark.parametrize("kv", ["i8", "f16"])
@pytest.mark.parametrize("act,H,KVH,hd,n,new", [("f32", 16, 16, 128, 4500, 1), ("bf16", 32, 4, 128, 9000, 1),
                                                ("f16", 8, 1, 64, 20011, 3), ("f32", 4, 1, 128, 3000, 40)])
def test_attention_of_a_long_context(kv, act, H, KVH, hd, n, new):
    rng = np.random.default_rng(n)
    rig = Rig(H, KVH, hd, 64, kv, act, 400, 400)
    pages = tables(rng, 400, 400, [-(-(n + new) // 64)])
    fill(rig, rng, [n], pages)
    rig.append([n], [new], pages, normal(rng, new, KVH, hd), normal(rng, new, KVH, hd))
    rig.check_attention([n], [new], pages, normal(rng, new, H, hd, scale=2.0))


@pytest.mark.parametrize("kv", ["i8", "f16"])
def test_prompt(kv):
    rng = np.random.default_rng(11)
    rig = Rig(8, 2, 128, 32, kv, "bf16", 60, 30)
    pages = tables(rng, 60, 30, [21, 16])
    new = [650, 509]
    rig.append([0, 0], new, pages, normal(rng, 1159, 2, 128), normal(rng, 1159, 2, 128))
    rig.check_attention([0, 0], new, pages, normal(rng, 1159, 8, 128))


# enough rows that a block takes many of them at a time
@pytest.mark.parametrize("kv", ["i8", "f16"])
@pytest.mark.parametrize("act,hd,lens,new", [
    ("f32", 64, [0, 300], [700, 331]), ("bf16", 128, [70, 0, 5], [601, 1, 300]),
    ("f16", 96, [129], [1000]), ("bf16", 48, [0], [1025]), ("f32", 256, [0, 33], [500, 200]),
    ("f16", 160, [64], [600])])
def test_many_rows(kv, act, hd, lens, new):
    rng = np.random.default_rng(hd)
    held = [-(-(a + b) // 32) for a, b in zip(lens, new)]
    rig = Rig(24, 24, hd, 32, kv, act, sum(held), max(held))
    pages = tables(rng, rig.n_pages, rig.max_pages, held)
    if any(lens):
        fill(rig, rng, lens, pages)
    N = sum(new)
    rig.append(lens, new, pages, normal(rng, N, 24, hd), normal(rng, N, 24, hd))
    rig.check_attention(lens, new, pages, normal(rng, N, 24, hd, scale=2.0), every=7)


@pytest.mark.parametrize("kv", ["i8", "f16"])
def test_many_rows_and_a_missing_page(kv):
    rng = np.random.default_rng(20)
    rig = Rig(24, 24, 64, 16, kv, "f32", 80, 70)
    pages = tables(rng, 80, 70, [70])
    pages[0, [3, 40]] = -1, 80
    x = normal(rng, 1100, 24, 64), normal(rng, 1100, 24, 64)
    rig.append([0], [1100], pages, *x)
    rig.check_attention([0], [1100], pages, normal(rng, 1100, 24, 64), every=5)


@pytest.mark.parametrize("bad", [np.inf, np.nan])
def test_many_rows_and_nonfinite_values(bad):
    rng = np.random.default_rng(21)
    rig = Rig(24, 24, 64, 16, "f16", "f32", 80, 70)
    pages = tables(rng, 80, 70, [70])
    k, v, q = (normal(rng, 1100, 24, 64) for _ in range(3))
    rig.append([0], [1100], pages, k, v)
    clean = rig.attention([0], [1100], pages, q)
    for tok, head, d in ((37, 3, 5), (511, 3, 63), (512, 7, 0), (1090, 23, 33)):
        v[tok, head, d] = bad
    rig.append([0], [1100], pages, k, v)
    got = rig.attention([0], [1100], pages, q)
    want = clean.copy()
    for tok, head, d in ((37, 3, 5), (511, 3, 63), (512, 7, 0), (1090, 23, 33)):
        assert not np.isfinite(got[tok:, head, d]).any()
        got[tok:, head, d] = want[tok:, head, d]
    np.testing.assert_array_equal(got, want)


# heads enough that every one has a block of many rows to itself, whatever its
# size: tiles of 256 or 128 rows that end early, one after another, over contexts
# of one step and of many
@pytest.mark.parametrize("kv", ["i8", "f16"])
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd,lens,new", [(32, [0], [17]), (64, [33, 0], [40, 300]), (96, [0], [150]),
                                         (128, [0, 75], [18, 290]), (160, [5], [140]), (192, [0], [64]),
                                         (256, [0, 61], [131, 3])])
def test_many_heads_of_many_rows(kv, act, hd, lens, new):
    H, rng = 200, np.random.default_rng(hd + len(act))
    held = [-(-(a + b) // 32) for a, b in zip(lens, new)]
    rig = Rig(H, H, hd, 32, kv, act, sum(held), max(held))
    pages = tables(rng, rig.n_pages, rig.max_pages, held)
    if any(lens):
        fill(rig, rng, lens, pages)
    N = sum(new)
    rig.append(lens, new, pages, normal(rng, N, H, hd), normal(rng, N, H, hd))
    rig.check_attention(lens, new, pages, normal(rng, N, H, hd, scale=2.0), every=29)


@pytest.mark.parametrize("kv", ["i8", "f16"])
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_many_heads_and_a_missing_page(kv, act, hd):
    H, rng = 200, np.random.default_rng(hd)
    rig = Rig(H, H, hd, 16, kv, act, 20, 18)
    pages = tables(rng, 20, 18, [18])
    pages[0, [0, 3, 10]] = -1, 20, -5
    x = normal(rng, 280, H, hd), normal(rng, 280, H, hd)
    rig.append([0], [280], pages, *x)
    rig.check_attention([0], [280], pages, normal(rng, 280, H, hd), every=31)


@pytest.mark.parametrize("bad", [np.inf, np.nan])
@pytest.mark.parametrize("act,hd", [("f32", 64), ("f16", 128), ("bf16", 128), ("f16", 256)])
def test_many_heads_and_nonfinite_values(bad, act, hd):
    H, rng = 200, np.random.default_rng(hd)
    rig = Rig(H, H, hd, 16, "f16", act, 20, 18)
    pages = tables(rng, 20, 18, [18])
    k, v, q = (normal(rng, 280, H, hd) for _ in range(3))
    rig.append([0], [280], pages, k, v)
    clean = rig.attention([0], [280], pages, q)
    at = ((37, 3, 5), (63, 3, 63), (64, 7, 0), (130, 199, 33), (279, 11, 12))
    for tok, head, d in at:
        v[tok, head, d] = bad
    rig.append([0], [280], pages, k, v)
    got = rig.attention([0], [280], pages, q)
    for tok, head, d in at:
        assert not np.isfinite(got[tok:, head, d]).any()
        got[tok:, head, d] = clean[tok:, head, d]
    np.testing.assert_array_equal(got, clean)


@pytest.mark.parametrize("kv", ["i8", "f16"])
@pytest.mark.parametrize("new", [1, 30])
def test_missing_pages(kv, new):
    """Ids outside the pool: nothing is written there, the keys are not there,
    and a row without any key is zeros."""
    rng = np.random.default_rng(2)
    rig = Rig(4, 2, 64, 16, kv, "f32", 30, 10)
    pages = tables(rng, 30, 10, [10, 10, 10])
    lens = [100, 70, 50]
    pages[0, [0, 3]] = -1, 30
    pages[1, :] = [2**31 - 1, -2**31, -1, 30, 31, -7, 100, 1000, -1, -1]
    pages[2, 3] = -5
    fill(rig, rng, lens, pages)
    rig.append(lens, [new] * 3, pages, normal(rng, 3 * new, 2, 64), normal(rng, 3 * new, 2, 64))
    rig.check_held([n + new for n in lens], pages)
    got = rig.check_attention(lens, [new] * 3, pages, normal(rng, 3 * new, 4, 64))
    assert not got[new:2 * new].any()


@pytest.mark.parametrize("kv", ["i8", "f16"])
def test_past_the_table(kv):
    """Tokens past the page table are dropped, their rows left as they were."""
    rng = np.random.default_rng(4)
    rig = Rig(4, 2, 64, 16, kv, "f32", 8, 2)
    pages = tables(rng, 8, 2, [2, 2])
    fill(rig, rng, [20, 7], pages)
    lens, new = [20, 32], [20, 3]
    k, v, q = (normal(rng, 23, h, 64) for h in (2, 2, 4))
    rig.append(lens, new, pages, k, v)
    rig.check_held([32, 7], pages)
    got = rig.attention(lens, new, pages, q)
    assert (got[12:] == 7).all()
    rig.check_attention([20, 32], [12, 0], pages, q[:12], got=got[:12])


def test_counts_that_do_not_fit():
    """starts that fall, or pass n_rows, max_new too small, negative lengths:
    rows inside the call's, positions inside the table."""
    rng = np.random.default_rng(6)
    rig = Rig(4, 2, 64, 16, "i8", "f32", 8, 2)
    pages = tables(rng, 8, 2, [2, 2, 2])
    fill(rig, rng, [10, 10, 10], pages)
    q = normal(rng, 6, 4, 64)
    b, keep = rig.batch([10, 10, 10], [2, 2, 2], pages)
    keep[0].upload(np.array([0, 4, -3, 90], np.int32))
    keep[1].upload(np.array([-5, 2**31 - 1, 3], np.int32))
    new = [2, 2, 2]
    rig.append([0] * 3, new, pages, normal(rng, 6, 2, 64), normal(rng, 6, 2, 64), batch=(b, keep))
    rig.attention([0] * 3, new, pages, q, batch=(b, keep))  # ends, inside its buffers


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("offset", [1, 3])
def test_unaligned_rows(act, offset):
    """Operands aligned to their elements only, rows an odd distance apart."""
    rng = np.random.default_rng(7)
    rig = Rig(4, 2, 96, 16, "i8", act, 20, 6)
    pages = tables(rng, 20, 6, [6, 6])
    lens, new = [30, 0], [1, 40]
    fill(rig, rng, lens, pages)
    k, v, q = normal(rng, 41, 2, 96), normal(rng, 41, 2, 96), normal(rng, 41, 4, 96)
    rig.append(lens, new, pages, k, v)
    aligned = rig.attention(lens, new, pages, q)
    np.testing.assert_array_equal(aligned, rig.attention(lens, new, pages, q, offset=offset))
    # the same tokens again, from unaligned rows: the same cache
    before = rig.read([0, 0], [31, 40], pages)
    row = 192
    rows = np.zeros((41, 2 * row + 5), to_bits(k, act).dtype)
    rows[:, :row], rows[:, row:2 * row] = to_bits(k.reshape(41, row), act), to_bits(v.reshape(41, row), act)
    flat = np.concatenate([np.zeros(offset, rows.dtype), rows.reshape(-1)])
    buf = hip.DeviceBuffer(flat.nbytes).upload(flat)
    b, keep = rig.batch(lens, new, pages)
    p, it = buf.ptr + offset * rows.itemsize, rows.itemsize
    L.kv_append_dev(rig.desc, rig.pool, b, p, 2 * row + 5, p + row * it, 2 * row + 5, rig.rope.ptr,
                    rig.stream.ptr)
    out = hip.DeviceBuffer(71 * (row + 1) * it + it), hip.DeviceBuffer(71 * (row + 1) * it + it)
    b, keep2 = rig.batch([0, 0], [31, 40], pages)
    L.kv_read_dev(rig.desc, rig.pool, b, out[0].ptr + it, row + 1, out[1].ptr + it, row + 1,
                  rig.stream.ptr)
    rig.stream.synchronize()
    for o, want in zip(out, before):
        got = o.download(np.empty(71 * (row + 1) + 1, rows.dtype))[1:].reshape(71, row + 1)[:, :row]
        np.testing.assert_array_equal(from_bits(got, act).reshape(want.shape), want)


def test_i8_of_extreme_values():
    """Infinities, NaN, zeros, the largest and smallest f32: finite codes, the
    reference's."""
    rng = np.random.default_rng(8)
    rig = Rig(2, 2, 32, 16, "i8", "f32", 8, 2, rope=False)
    pages = tables(rng, 8, 2, [2, 2, 2])
    k, v = normal(rng, 30, 2, 32), normal(rng, 30, 2, 32)
    k[0, 0, 3], k[1, 0, 4], k[2, 1, 5] = np.inf, -np.inf, np.nan
    v[10:20] = 0
    v[12, 0, 0] = np.inf
    k[20:, 0] *= np.float32(3e38) / np.abs(k[20:, 0]).max()
    k[20:, 1] *= np.float32(1e-40)
    v[20:, 0] = 1e-45
    rig.append([0, 0, 0], [10, 10, 10], pages, k, v)
    rig.check_held([10, 10, 10], pages)


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("which", ["k", "v"])
def test_f16_nonfinite_stays_with_its_readers(which, bad, act):
    """A key or value that is not finite reaches the rows that see it, and no
    earlier row of the same tile."""
    rng = np.random.default_rng(9)
    rig = Rig(4, 2, 64, 16, "f16", act, 20, 8)
    pages = tables(rng, 20, 8, [8])
    T, at = 90, 37
    x = {"k": normal(rng, T, 2, 64), "v": normal(rng, T, 2, 64)}
    q = normal(rng, T, 4, 64)
    rig.append([0], [T], pages, x["k"], x["v"])
    clean = rig.attention([0], [T], pages, q)
    x[which][at, 1, 5] = bad
    rig.append([0], [T], pages, x["k"], x["v"])
    got = rig.attention([0], [T], pages, q)
    np.testing.assert_array_equal(got[:at], clean[:at])
    np.testing.assert_array_equal(got[:, :2], clean[:, :2])
    if which == "v":
        assert not np.isfinite(got[at:, 2:, 5]).any()
        keep = np.arange(64) != 5
        np.testing.assert_array_equal(got[:, 2:, keep], clean[:, 2:, keep])
    elif np.isnan(bad):
        assert np.isnan(got[at:, 2:]).all()
    # one token alone, after it
    one = rig.attention([T - 1], [1], pages, q[T - 1:])
    assert np.isfinite(one[:, :2]).all() and not np.isfinite(one[:, 2:, 5]).any() or which == "k"


@pytest.mark.parametrize("kv", ["i8", "f16"])
@pytest.mark.parametrize("bad", [np.inf, np.nan])
def test_nonfinite_query(kv, bad):
    rng = np.random.default_rng(10)
    rig = Rig(4, 2, 64, 16, kv, "f32", 20, 8)
    pages = tables(rng, 20, 8, [8])
    rig.append([0], [50], pages, normal(rng, 50, 2, 64), normal(rng, 50, 2, 64))
    q = normal(rng, 50, 4, 64)
    clean = rig.attention([0], [50], pages, q)
    q[20, 1, 7] = bad
    got = rig.attention([0], [50], pages, q)
    assert np.isnan(got[20, 1]).all()
    got[20, 1] = clean[20, 1]
    np.testing.assert_array_equal(got, clean)


@pytest.mark.parametrize("kv", ["i8", "f16"])
def test_sizes_of_q(kv):
    """Queries far outside f16's range, and rows of zeros."""
    rng = np.random.default_rng(12)
    rig = Rig(4, 2, 64, 16, kv, "f32", 20, 8)
    pages = tables(rng, 20, 8, [8])
    rig.append([0], [50], pages, normal(rng, 50, 2, 64), normal(rng, 50, 2, 64))
    q = normal(rng, 50, 4, 64)
    q[3] = 0
    for s in (1e-30, 1e30):
        rig.check_attention([0], [50], pages, q * np.float32(s), scale=0.125 / s)


def test_offsets_past_32_bits():
    """The last pages of a pool of more than 4 GiB each of keys and values."""
    rng = np.random.default_rng(13)
    KVH, hd, page, n_pages = 8, 128, 256, 9000
    rig = Rig.__new__(Rig)
    small = Rig(16, KVH, hd, page, "f16", "f32", 8, 4)
    rig.__dict__.update(small.__dict__)
    rig.n_pages = n_pages
    rig.desc = L.KvDesc(16, KVH, hd, page, n_pages, 4, L.TYPE_F16, L.TYPE_F32, L.ROPE_ABSOLUTE)
    n, _ = L.kv_sizes(rig.desc)
    assert n > 4 << 30
    rig.bufs = [hip.DeviceBuffer(n), hip.DeviceBuffer(n)]
    rig.pool = L.KvPool(rig.bufs[0].ptr, rig.bufs[1].ptr, None)
    pages = np.array([[n_pages - 1, n_pages - 4, n_pages - 2, 0]], np.int32)
    # the reference holds the same pages under small numbers
    names = np.array([[7, 4, 6, 0]], np.int32)
    k, v, q = normal(rng, 600, KVH, hd), normal(rng, 600, KVH, hd), normal(rng, 600, 16, hd)
    with pytest.raises(AssertionError):  # the reference under its own names holds nothing yet
        np.testing.assert_array_equal(rig.ref.values(0, names[0], 600)[0], k.astype(np.float64))
    real = rig.ref.append
    rig.ref.append = lambda p, *a: real(names[0], *a)
    rig.append([0], [600], pages, k, v)
    got = rig.attention([0], [600], pages, q)
    rig.check_attention([0], [600], names, q, got=got)
    want = rig.ref.values(1, names[0], 600)[0]
    np.testing.assert_array_equal(rig.read([0], [600], pages)[1], want)
    for b in rig.bufs:
        b.free()


@pytest.mark.parametrize("kv", ["i8", "f16"])
def test_two_streams(kv):
    """Two calls at once, a workspace each."""
    rng = np.random.default_rng(14)
    rigs = [Rig(8, 2, 128, 16, kv, "f32", 200, 100) for _ in range(2)]
    pages = tables(rng, 200, 100, [100])
    want, jobs = [], []
    for rig in rigs:
        fill(rig, rng, [1500], pages)
        q = normal(rng, 1, 8, 128)
        want.append(rig.check_attention([1499], [1], pages, q))
        b, keep = rig.batch([1499], [1], pages)
        qb, ob = hip.DeviceBuffer(q.nbytes).upload(q), hip.DeviceBuffer(q.nbytes)
        n = L.kv_attention_workspace(rig.desc, b)
        jobs.append((rig, b, keep, qb, ob, hip.DeviceBuffer(max(n, 16)), n))
    for _ in range(20):
        for rig, b, _k, qb, ob, ws, n in jobs:
            L.kv_attention_dev(rig.desc, rig.pool, b, qb.ptr, 1024, rig.rope.ptr, 128 ** -0.5, ob.ptr,
                               1024, ws.ptr, n, rig.stream.ptr)
    for (rig, *_, ob, ws, n), w in zip(jobs, want):
        rig.stream.synchronize()
        np.testing.assert_array_equal(ob.download(np.empty((1, 8, 128), np.float32)), w)


def test_a_captured_step():
    """A decode step (append, attention, log probabilities) captured once and
    replayed as lengths, tokens and queries move on, against eager calls."""
    rng = np.random.default_rng(15)
    rig = Rig(8, 2, 64, 16, "i8", "f32", 40, 12)
    twin = Rig(8, 2, 64, 16, "i8", "f32", 40, 12)
    pages = tables(rng, 40, 12, [12, 12])
    lens = np.array([30, 5], np.int32)
    state = rng.bit_generator.state
    for r in (rig, twin):
        rng.bit_generator.state = state
        fill(r, rng, list(lens), pages)
    d_lens, d_pages = hip.DeviceBuffer(8), hip.DeviceBuffer(pages.nbytes).upload(pages)
    kv, q = hip.DeviceBuffer(2 * 256 * 4), hip.DeviceBuffer(2 * 512 * 4)
    results = [np.empty((2, 512), np.float32), np.empty(2, np.float32), np.empty((2, 4), np.int32),
               np.empty((2, 4), np.float32)]
    bufs = [hip.DeviceBuffer(r.nbytes) for r in results]
    out, ent, ids, lps = (b.ptr for b in bufs)
    b = L.KvBatch(2, 2, 1, None, d_lens.ptr, d_pages.ptr)
    n = max(L.kv_attention_workspace(rig.desc, b), L.logprobs_workspace(L.TYPE_F32, 2, 512, 0, 4), 16)
    ws = [hip.DeviceBuffer(n) for _ in range(2)]

    def step(r, w):
        st = r.stream.ptr
        L.kv_append_dev(r.desc, r.pool, b, kv.ptr, 256, kv.ptr + 512, 256, r.rope.ptr, st)
        L.kv_attention_dev(r.desc, r.pool, b, q.ptr, 512, r.rope.ptr, 0.125, out, 512, w.ptr, n, st)
        L.logprobs_dev(L.TYPE_F32, out, 512, 2, 512, None, 0, None, ent, 4, ids, lps, w.ptr, n, st)

    g = Graph(rig.stream, lambda: step(rig, ws[0]))
    for i in range(6):
        d_lens.upload(lens)
        kv.upload(normal(rng, 2, 256, scale=1 + i))
        q.upload(normal(rng, 2, 512))
        g.replay()
        rig.stream.synchronize()
        got = [x.download(np.empty_like(r)) for x, r in zip(bufs, results)]
        bufs[0].upload(np.zeros((2, 512), np.float32))
        step(twin, ws[1])
        twin.stream.synchronize()
        for a, x, r in zip(got, bufs, results):
            np.testing.assert_array_equal(a, x.download(r))
        assert got[0].any()
        lens += 1
    g.close()


def test_the_activation_types_agree_on_exact_values():
    """Values that every type holds: the same cache from each."""
    rng = np.random.default_rng(16)
    held = []
    for act in ACTS:
        rig = Rig(2, 2, 64, 16, "i8", act, 8, 4, rope=False)
        pages = np.arange(4, dtype=np.int32)[None]
        x = np.random.default_rng(17).integers(-8, 9, (50, 2, 64)).astype(np.float32)
        rig.append([0], [50], pages, x, x[::-1].copy())
        rig.check_held([50], pages)
        held.append([rig.ref.data.copy(), rig.ref.scale.copy()])
    for h in held[1:]:
        np.testing.assert_array_equal(h[0], held[0][0])
        np.testing.assert_array_equal(h[1], held[0][1])
