"""The paged cache's and the log probabilities' host side: sizes, the rope
table and every refusal, before any device work."""
import ctypes as C

import numpy as np
import pytest

import leafcutterllm_amd as L
from leafcutterllm_amd import _lib

FAKE = 1 << 20  # never dereferenced: each check comes before the device


def desc(**kw):
    d = dict(n_head=8, n_kv_head=2, head_dim=64, page_tokens=16, n_pages=10, max_pages=4,
             kv_type=L.TYPE_I8, act_type=L.TYPE_F32, rope_positions=L.ROPE_ABSOLUTE)
    d.update(kw)
    return L.KvDesc(**d)


def batch(**kw):
    b = dict(n_seq=2, n_rows=5, max_new=3, starts=FAKE, lens=FAKE, pages=FAKE)
    b.update(kw)
    return L.KvBatch(**b)


def pool(**kw):
    p = dict(k=FAKE, v=FAKE, scale=FAKE)
    p.update(kw)
    return L.KvPool(**p)


def append(d=None, p=None, b=None, k=FAKE, ldk=128, v=FAKE, ldv=128, rope=FAKE):
    L.kv_append_dev(d or desc(), p or pool(), b or batch(), k, ldk, v, ldv, rope)


def read(d=None, p=None, b=None, k=FAKE, ldk=128, v=FAKE, ldv=128):
    L.kv_read_dev(d or desc(), p or pool(), b or batch(), k, ldk, v, ldv)


def attention(d=None, p=None, b=None, q=FAKE, ldq=512, rope=FAKE, scale=0.125, out=FAKE, ldo=512,
              ws=FAKE, n=1 << 40):
    L.kv_attention_dev(d or desc(), p or pool(), b or batch(), q, ldq, rope, scale, out, ldo, ws, n)


def refused(status, f, *a, **kw):
    with pytest.raises(L.LcmoeError) as e:
        f(*a, **kw)
    assert e.value.status == status and L.lib().lcmoe_last_error()


def test_sizes():
    # 10 pages x 2 heads x 16 tokens x 64 dims
    assert L.kv_sizes(desc()) == (20480, 160)
    assert L.kv_sizes(desc(kv_type=L.TYPE_F16)) == (40960, 0)
    assert L.kv_sizes(desc(head_dim=80)) == (20480 * 96 // 64, 160)  # held as 96 dims
    assert L.kv_sizes(desc(n_pages=2**31 - 1, n_kv_head=8, page_tokens=256)) == \
        ((2**31 - 1) * 8 * 256 * 64, (2**31 - 1) * 64)


@pytest.mark.parametrize("field,value,status", [
    ("n_head", 0, 1), ("n_head", 7, 1), ("n_head", 65536 * 2, 1), ("n_kv_head", 0, 1),
    ("n_kv_head", 3, 1), ("head_dim", 8, 1), ("head_dim", 72, 1), ("head_dim", 272, 1),
    ("page_tokens", 8, 1), ("page_tokens", 48, 1), ("page_tokens", 512, 1), ("page_tokens", -16, 1),
    ("n_pages", 0, 1), ("max_pages", 0, 1), ("max_pages", 2**31 // 16, 1), ("kv_type", 0, 2),
    ("kv_type", 8, 2), ("act_type", 24, 2), ("act_type", 12, 2), ("rope_positions", 2, 1)])
def test_desc_refusals(field, value, status):
    d = desc(**{field: value})
    refused(status, L.kv_sizes, d)
    refused(status, append, d)
    refused(status, read, d)
    refused(status, attention, d)
    refused(status, L.kv_attention_workspace, d, batch())


@pytest.mark.parametrize("kw", [
    dict(n_seq=-1), dict(n_rows=-1), dict(max_new=-1), dict(lens=None), dict(pages=None),
    dict(starts=None), dict(starts=None, n_rows=7), dict(lens=FAKE + 2), dict(pages=FAKE + 1),
    dict(starts=FAKE + 3), dict(n_seq=1 << 21), dict(n_rows=(1 << 30) + 1)])
def test_batch_refusals(kw):
    for f in (append, read, attention):
        refused(1, f, b=batch(**kw))


def test_operand_refusals():
    for f in (append, read, attention):
        refused(1, f, p=pool(k=None))
        refused(1, f, p=pool(v=None))
        refused(1, f, p=pool(scale=None))
        refused(1, f, p=pool(scale=FAKE + 4))
        refused(1, f, p=pool(k=FAKE + 8))
        refused(1, f, p=pool(v=FAKE + 2))
    for f in (append, read):
        refused(1, f, k=None)
        refused(1, f, v=None)
        refused(1, f, ldk=127)
        refused(1, f, ldv=0)
        refused(1, f, k=FAKE + 2)
        refused(1, f, desc(act_type=L.TYPE_BF16), v=FAKE + 1)
    refused(1, append, rope=FAKE + 4)
    refused(1, attention, rope=FAKE + 4)
    refused(1, attention, q=None)
    refused(1, attention, out=None)
    refused(1, attention, ldq=511)
    refused(1, attention, ldo=511)
    refused(1, attention, q=FAKE + 3)
    for s in (0.0, -1.0, float("inf"), float("nan")):
        refused(1, attention, scale=s)


def test_workspace_refusals():
    # a long document's token: several blocks share a head, so partials go
    # through the workspace
    d, b = desc(max_pages=8192, n_pages=8192), batch(n_seq=1, n_rows=1, max_new=1)
    n = L.kv_attention_workspace(d, b)
    assert n > 0
    # it depends on the sizes alone
    assert n == L.kv_attention_workspace(d, L.KvBatch(n_seq=1, n_rows=1, max_new=1))
    refused(1, attention, d, b=b, ws=None)
    refused(1, attention, d, b=b, n=n - 1)
    refused(1, attention, d, b=b, ws=FAKE + 8, n=n)
    assert L.lib().lcmoe_kv_attention_workspace(C.byref(d), C.byref(b), None) == 1


def test_attention_too_many_rows():
    refused(1, attention, b=batch(n_rows=(1 << 30) - 1, max_new=3))
    refused(1, L.kv_attention_workspace, desc(), batch(n_rows=(1 << 30) - 1, max_new=3))


@pytest.mark.parametrize("kw", [dict(n_seq=0, n_rows=0, max_new=0), dict(n_rows=0), dict(max_new=0)])
def test_nothing_to_do(kw):
    """No rows: no operand is looked at, and no device needed."""
    b = batch(starts=FAKE, **kw)
    L.kv_append_dev(desc(), pool(k=None), b, None, 0, None, 0)
    L.kv_read_dev(desc(), pool(k=None), b, None, 0, None, 0)
    L.kv_attention_dev(desc(), pool(k=None), b, None, 0, None, 1.0, None, 0, None, 0)
    assert L.kv_attention_workspace(desc(), b) == 0


def test_null_structs():
    lib = L.lib()
    append(b=batch(n_rows=0))  # binds
    d, p, b = desc(), pool(), batch()
    for args in ((None, p, b), (d, None, b), (d, p, None)):
        assert lib.lcmoe_kv_append_dev(*args, FAKE, 128, FAKE, 128, None, None) == 1
        assert lib.lcmoe_kv_read_dev(*args, FAKE, 128, FAKE, 128, None) == 1
        assert lib.lcmoe_kv_attention_dev(*args, FAKE, 512, None, 1.0, FAKE, 512, FAKE, 1 << 40,
                                          None) == 1


@pytest.mark.parametrize("theta,hd", [(10000.0, 128), (500000.0, 64), (10000.0, 16)])
def test_rope_table(theta, hd):
    t = L.rope_table(theta, hd, 4099).astype(np.float64)
    a = np.arange(4099)[:, None] * np.float64(np.float32(theta)) ** (-np.arange(0, hd, 2) / hd)
    # the angle to 2^-52 of itself, a cosine rounded once
    tol = 2.0**-24 + np.abs(a) * 2.0**-51
    assert np.all(np.abs(t[..., 0] - np.cos(a)) <= tol)
    assert np.all(np.abs(t[..., 1] - np.sin(a)) <= tol)


def test_rope_table_refusals():
    for theta, hd, n in ((0.0, 64, 4), (float("nan"), 64, 4), (float("inf"), 64, 4), (1e4, 3, 4),
                         (1e4, 0, 4), (1e4, 64, -1)):
        refused(1, L.rope_table, theta, hd, n)
    assert L.rope_table(1e4, 64, 0).shape == (0, 32, 2)
    assert L.lib().lcmoe_rope_table(1e4, 64, 1, None) == 1


def lp(type=L.TYPE_F32, x=FAKE, ld=100, rows=3, vocab=100, given=FAKE, n_given=1, glp=FAKE,
       ent=FAKE, top=2, tid=FAKE, tlp=FAKE, ws=FAKE, n=1 << 40):
    L.logprobs_dev(type, x, ld, rows, vocab, given, n_given, glp, ent, top, tid, tlp, ws, n)


@pytest.mark.parametrize("kw,status", [
    (dict(type=L.TYPE_I8), 2), (dict(type=L.TYPE_Q4_K), 2), (dict(rows=-1), 1), (dict(vocab=0), 1),
    (dict(ld=99), 1), (dict(n_given=-1), 1), (dict(n_given=65537), 1), (dict(top=-1), 1),
    (dict(top=33), 1), (dict(x=None), 1), (dict(given=None), 1), (dict(glp=None), 1),
    (dict(tid=None), 1), (dict(tlp=None), 1), (dict(x=FAKE + 2), 1), (dict(given=FAKE + 1), 1),
    (dict(ent=FAKE + 2), 1), (dict(type=L.TYPE_BF16, x=FAKE + 1), 1),
    (dict(vocab=2**30 + 1, ld=2**30 + 1), 1), (dict(vocab=2**31 - 1, ld=2**31), 1)])
def test_logprobs_refusals(kw, status):
    refused(status, lp, **kw)


def test_logprobs_workspace_and_nothing():
    n = L.logprobs_workspace(L.TYPE_F32, 1, 1_000_000, 1, 5)
    assert n > 0
    big = dict(rows=1, vocab=1_000_000, ld=1_000_000, top=5)
    refused(1, lp, ws=None, **big)
    refused(1, lp, n=n - 1, **big)
    refused(1, lp, ws=FAKE + 8, n=n, **big)
    refused(2, L.logprobs_workspace, 7, 1, 10, 1, 1)
    refused(1, L.logprobs_workspace, 0, 1, 0, 1, 1)
    L.logprobs_dev(L.TYPE_F32, None, 10, 0, 10, None, 1, None, None, 1, None, None, None, 0)
    L.logprobs_dev(L.TYPE_F32, None, 10, 3, 10, None, 0, None, None, 0, None, None, None, 0)
    out = L.logprobs(np.zeros((0, 10), np.float32), np.zeros((0, 2), np.int32), 3)
    assert [x.shape for x in out] == [(0, 2), (0,), (0, 3), (0, 3)]


def test_logprobs_python_refusals():
    x = np.zeros((2, 10), np.float32)
    for args in ((x.astype(np.float64),), (np.zeros((2, 2, 2), np.float32),),
                 (x, np.zeros((3, 1), np.int32)), (x, None, 33), (x, None, -1)):
        with pytest.raises(L.LcmoeError) as e:
            L.logprobs(*args)
        assert _lib.STATUS[e.value.status] == "LCMOE_ERR_INVALID_ARG"


def test_paged_models_refusals():
    """What lcmoe_model_create_paged and lcmoe_model_score refuse before any
    device work."""
    from leafcutterllm_amd.configs import ModelConfig, small_config, synth_model

    mc = ModelConfig("tiny", 1, 4, 2, 64, 32, 10000.0,
                     small_config("m", 256, 256, 8, 2, L.ROUTE_SOFTMAX, L.TYPE_Q4_K, L.TYPE_Q4_K))
    w = synth_model(mc, seed=1)
    for kv in ((L.TYPE_I8, 24, 0), (L.TYPE_I8, 0, 0), (L.TYPE_I8, -16, 0), (L.TYPE_I8, 512, 0),
               (L.TYPE_F16, 16, -1), (L.TYPE_F32, 16, 0), (L.TYPE_Q8_0, 16, 0)):
        with pytest.raises(L.LcmoeError) as e:
            L.Model(mc.desc(2, 16, 32), w, *kv)
        assert _lib.STATUS[e.value.status] in ("LCMOE_ERR_INVALID_ARG", "LCMOE_ERR_UNSUPPORTED"), kv
    t = np.zeros(4, np.int32)
    lib = L.lib()
    assert lib.lcmoe_model_score(None, t.ctypes.data, None, 1, 4, None, None, 0, None, None) == 1
