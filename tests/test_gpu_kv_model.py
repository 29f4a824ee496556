"""GPU: the decoder over a paged cache (lcmoe_model_create_paged) and its
scoring of texts (lcmoe_model_score), against the oracle's engine with its
cache held in pages as include/lcmoe.h defines them.

Bar: that of the unpaged model for f16 pages, last-token logits within 1e-3
relative L2 of the oracle's and the same greedy ids.  8-bit codes widen what the
two engines' keys and values differ by before the cache: a relative difference
e moves a value x by 127 e |x| / max steps, which is the chance that its code is
another, by one step.  Over values of rms r max that is an error of
sqrt(127 e r) steps of 127 r: with e = 1e-3, the bar itself, and r = 0.31
(normal values, the largest of a page's 1024 being 3.2 sigma) sqrt(0.039) / 39 =
5e-3 of keys and values, 5e-3 of the logits at most where the attention's
output is no more than the residual it is added to.  So 6e-3 in all."""
import numpy as np
import pytest

import lcengine as E
import lcoracle as O
import leafcutterllm_amd as L
from kv_ref import KVS, RefCache
from leafcutterllm_amd import _lib
from leafcutterllm_amd.configs import ModelConfig, small_config, synth_model
from test_gpu_engine import LOGIT_TOL
from test_oracle_engine import TINY, rel, spec

pytestmark = pytest.mark.gpu

TOL = {None: LOGIT_TOL, "f16": LOGIT_TOL, "i8": 6e-3}


class PagedEngine(E.RefEngine):
    """RefEngine with RefCache pages; forward keeps every token's logits in
    self.rows."""

    def __init__(self, s, w, kv, page):
        self.kv, self.page = kv, page
        super().__init__(s, w, threads=8)

    def clear(self):
        s = self.s
        self.n = 0
        self.cache = [RefCache(64, s.n_kv_head, s.head_dim, self.page, self.kv) for _ in self.layers]

    def forward(self, tokens):
        s = self.s
        H, KVH, hd, T, pages = s.n_head, s.n_kv_head, s.head_dim, len(tokens), list(range(64))
        hidden = np.stack([self.embed[t] if 0 <= t < s.vocab else np.zeros(s.d_model, np.float32)
                           for t in tokens])
        pos0 = self.n if s.rope_positions == E.ROPE_ABSOLUTE else 0
        for c, p, lw in zip(self.cache, self.layers, self.w["layers"]):
            x = O.rms_norm(hidden, p["attn_norm"], s.eps)
            q = O.rope(self._mm(x, p["wq"]), H, hd, s.rope_theta, pos0)
            k = O.rope(self._mm(x, p["wk"]), KVH, hd, s.rope_theta, pos0)
            c.append(pages, self.n, k.astype(np.float64).reshape(T, KVH, hd),
                     self._mm(x, p["wv"]).astype(np.float64).reshape(T, KVH, hd))
            k, v = [c.values(j, pages, self.n + T)[0].astype(np.float32).reshape(self.n + T, -1)
                    for j in (0, 1)]
            hidden = hidden + self._mm(O.attention_core(q, k, v, H, KVH, hd), p["wo"])
            x = O.rms_norm(hidden, p["ffn_norm"], s.eps)
            hidden = hidden + O.moe_forward(s.moe_desc, lw["moe"], x, threads=self.threads)["y"]
        self.n += T
        self.rows = self._mm(O.rms_norm(hidden, self.out_norm, s.eps), self.lm_head)
        return self.rows[-1]


def model(mc, w, mode, kv, page=16, n_pages=0, B=4, P=16, ctx=64):
    return L.Model(mc.desc(B, P, ctx, mode), w, KVS[kv], page, n_pages)


def assert_near(got, want, kv):
    e = rel(got, want.astype(np.float64))
    assert e < TOL[kv], e


def assert_same_greedy(got, ids, trace, kv):
    """The ids up to a step where the two are as near as the bar leaves open:
    two logits' difference moves by sqrt(2) times the L2 error."""
    for g, r, lg in zip(got, ids, trace):
        if g != r:
            lg = lg.astype(np.float64)
            assert lg[r] - lg[g] < 2**0.5 * TOL[kv] * np.linalg.norm(lg), (g, r)
            return
    assert len(got) == len(ids)


@pytest.mark.parametrize("kv", list(KVS))
@pytest.mark.parametrize("mode", [E.ROPE_PER_CALL, E.ROPE_ABSOLUTE])
def test_forward(kv, mode):
    w = synth_model(TINY, seed=7)
    ref = PagedEngine(spec(TINY, mode), w, kv, 16)
    calls = [[5, 17, 3, 95, 0, 60, 200], [11], [42], [7], [1, 2], list(range(16)), [3], [4, 5, 6]]
    with model(TINY, w, mode, kv) as m:
        for c in calls:
            assert_near(m.forward(np.array([c]))[0], ref.forward(c), kv)
        m.reset()
        ref.clear()
        assert_near(m.forward(np.array([[9, 8, 7]]))[0], ref.forward([9, 8, 7]), kv)


@pytest.mark.parametrize("kv", list(KVS))
@pytest.mark.parametrize("hd,H,KVH,page", [(160, 2, 1, 32), (256, 2, 2, 64), (96, 4, 1, 16)])
def test_heads_and_long_prompts(kv, hd, H, KVH, page):
    mc = ModelConfig("tiny-heads", 2, H, KVH, hd, 64, 10000.0,
                     small_config("tiny-heads", 256, 256, 8, 2, L.ROUTE_SOFTMAX_RENORM,
                                  L.TYPE_Q8_0, L.TYPE_Q8_0), attn_type=L.TYPE_Q8_0)
    w = synth_model(mc, seed=12)
    ref = PagedEngine(spec(mc, E.ROPE_ABSOLUTE), w, kv, page)
    with model(mc, w, E.ROPE_ABSOLUTE, kv, page, B=1, P=160, ctx=192) as m:
        for c in ([(7 * i + 3) % 64 for i in range(150)], [1], [2]):
            assert_near(m.forward(np.array([c]))[0], ref.forward(c), kv)


@pytest.mark.parametrize("kv", list(KVS))
def test_batch_of_unlike_lengths(kv):
    w = synth_model(TINY, seed=8)
    refs = [PagedEngine(spec(TINY, E.ROPE_ABSOLUTE), w, kv, 16) for _ in range(3)]
    with model(TINY, w, E.ROPE_ABSOLUTE, kv) as m:
        def both(rows):
            got = m.forward(np.array(rows))
            for g, r, ref in zip(got, rows, refs):
                assert_near(g, ref.forward(r), kv)
        both([[1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12]])
        both([[50, 60], [9, 9]])
        for i in range(5):
            both([[10 + i], [20 + i], [30 + i]])


@pytest.mark.parametrize("kv", list(KVS))
@pytest.mark.parametrize("mode", [E.ROPE_PER_CALL, E.ROPE_ABSOLUTE])
def test_generate(kv, mode):
    """Through the captured step, three sequences together, twice, then two;
    the eager steps' ids are the same, and a new call's pages are its own."""
    w = synth_model(TINY, seed=9)
    prompts = np.array([[3, 1, 4, 1, 5, 9], [2, 7, 1, 8, 2, 8], [90, 91, 92, 93, 94, 95]])
    n_new = 20
    refs = [PagedEngine(spec(TINY, mode), w, kv, 16).generate(list(p), n_new) for p in prompts]
    with model(TINY, w, mode, kv, n_pages=6) as m:
        for B in (3, 3, 2):
            out, n = m.generate(prompts[:B], n_new)
            assert np.all(n == n_new)
            for b in range(B):
                assert_same_greedy(list(out[b]), refs[b][0], refs[b][1], kv)
        m.set_decode_graph(False)
        assert np.array_equal(m.generate(prompts[:2], n_new)[0], out)


def test_pages_run_out():
    """A call that lacks pages changes nothing: the next one that fits goes on."""
    w, kv = synth_model(TINY, seed=10), "i8"
    ref = PagedEngine(spec(TINY, E.ROPE_PER_CALL), w, kv, 16)
    with model(TINY, w, E.ROPE_PER_CALL, kv, n_pages=2) as m:
        def short(f, *a):
            with pytest.raises(L.LcmoeError) as e:
                f(*a)
            assert _lib.STATUS[e.value.status] == "LCMOE_ERR_OUT_OF_MEMORY"
        assert_near(m.forward(np.array([[1] * 16]))[0], ref.forward([1] * 16), kv)
        short(m.forward, np.array([[2], [2], [2]]))
        assert_near(m.forward(np.array([[5] * 15]))[0], ref.forward([5] * 15), kv)
        assert_near(m.forward(np.array([[6]]))[0], ref.forward([6]), kv)
        for f in (m.forward, m.score):
            short(f, np.array([[7]]))
        short(m.generate, np.array([[1, 2], [3, 4], [5, 6]]), 3)
        ref.clear()
        assert_near(m.forward(np.array([[8, 9]]))[0], ref.forward([8, 9]), kv)
        m.reset()
        ref.clear()
        assert_near(m.forward(np.array([[3] * 16]))[0], ref.forward([3] * 16), kv)


def logprobs64(rows):
    x = rows.astype(np.float64)
    x -= x.max(-1, keepdims=True)
    return x - np.log(np.exp(x).sum(-1, keepdims=True))


@pytest.mark.parametrize("kv", [None, "f16", "i8"])
def test_score(kv):
    """Texts in several calls, 300 rows (more than are scored at once) in one,
    then a batch of single tokens."""
    w = synth_model(TINY, seed=13)
    refs = [PagedEngine(spec(TINY, E.ROPE_ABSOLUTE), w, kv or "f16", 16) for _ in range(2)]
    texts = np.array([[(7 * i + 5 * b + i * i) % TINY.vocab for i in range(311)] for b in range(2)])
    mk = model if kv else (lambda mc, w, mode, kv, **k: L.Model(mc.desc(k["B"], k["P"], k["ctx"], mode), w))
    with mk(TINY, w, E.ROPE_ABSOLUTE, kv, B=2, P=300, ctx=320) as m:
        for a, b in ((0, 1), (1, 10), (10, 310), (310, 311)):
            t = texts[:, a:b]
            targets = np.roll(texts, -1, 1)[:, a:b]
            lp, ent, ids, tlp = m.score(t, targets, 5)
            for i, ref in enumerate(refs):
                ref.forward(list(t[i]))
                want = logprobs64(ref.rows)
                # a logit off by the bar's whole L2 error, and the sum of them all
                tol = 2 * TOL[kv] * np.linalg.norm(ref.rows.astype(np.float64), axis=1)
                r = np.arange(b - a)
                assert np.all(np.abs(lp[i] - want[r, targets[i]]) < tol)
                # d entropy = -sum p (log p + entropy) d logit
                assert np.all(np.abs(ent[i] + (np.exp(want) * want).sum(1)) < tol * (1 + np.log(TINY.vocab)))
                assert np.all(np.abs(tlp[i] - np.sort(want, 1)[:, ::-1][:, :5]) < tol[:, None])
                assert np.all(np.abs(tlp[i] - np.take_along_axis(want, ids[i], 1)) < tol[:, None])


def test_score_beside_forward():
    """The defaults' targets; what is not wanted; caches go on as after forward."""
    w = synth_model(TINY, seed=14)
    text = np.array([[4, 8, 15, 16, 23, 42, 1000000, 7]])
    with model(TINY, w, E.ROPE_ABSOLUTE, "i8", B=1) as m:
        lp, ent, ids, tlp = m.score(text)
        assert ids.shape == (1, 8, 0) and lp[0, -1] == 0 and lp[0, 5] == 0 and (lp[0, :5] < 0).all()
        after = m.forward(np.array([[9]]))
        m.reset()
        full = m.forward(text)
        top = m.forward(np.array([[9]]))
        np.testing.assert_array_equal(after, top)
        m.reset()
        got = np.zeros((1, 8), np.float32)
        t = text.astype(np.int32)
        L.lib().lcmoe_model_score(m._h, t.ctypes.data, None, 1, 8, None, got.ctypes.data, 0, None, None)
        np.testing.assert_array_equal(got, ent)
        m.reset()
        best = m.score(text, n_top=1)[2][0, -1, 0]
        assert best == full[0].argmax()
        m.debug_fail_forward(0)
        for f in (m.score, m.score, m.forward):
            with pytest.raises(L.LcmoeError) as e:
                f(text)
            assert _lib.STATUS[e.value.status] == "LCMOE_ERR_STATE"
        m.reset()
        np.testing.assert_array_equal(m.score(text)[0], lp)
