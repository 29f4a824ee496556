"""The serving operators' cases: a paged K/V cache in f16 or in 8 bits, the
attention that reads it, and the log probabilities of the logits.

Each case is one call, as a serving program makes it with everything resident
on the GPU:

* `append`: a ragged batch's keys (rotated on the way) and values go into the
  pages of a cache.  In f16 the pools themselves are the result; in 8 bits the
  pages that the call touched are read back as the values they stand for
  (kv_append_dev, kv_read_dev);
* `attend`: causal attention of a ragged batch over such a cache, the queries
  rotated on the way (kv_attention_dev);
* `logprobs`: log probabilities of given tokens, the entropy and the top
  alternatives of rows of logits (logprobs_dev).

Where `own` is false, the same results come from elementary torch operations
on the same buffers.  A cache's page holds, per K/V head, units of 16 tokens;
`_k_places` and `_v_places` say where a unit keeps each value.
"""
from __future__ import annotations

import functools
import math

import torch

own = False
DEV = "cuda"
ACTS = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
THETA = 10000.0


def _append(name, B, T, ctx, KVH, hd, kv, page, act):
    return {"name": name, "kind": "append", "B": B, "T": T, "ctx": ctx, "H": KVH, "KVH": KVH,
            "hd": hd, "kv": kv, "page": page, "act": act}


def _attend(name, B, T, ctx, H, KVH, hd, kv, page, act):
    return {"name": name, "kind": "attend", "B": B, "T": T, "ctx": ctx, "H": H, "KVH": KVH,
            "hd": hd, "kv": kv, "page": page, "act": act}


def _logprobs(name, rows, vocab, pad, act, given, top):
    return {"name": name, "kind": "logprobs", "rows": rows, "vocab": vocab, "pad": pad,
            "act": act, "given": given, "top": top}


def listed():
    return [
        # a decode step of the decoder model's batch of 16: one token each
        _append("append-step", 16, 1, 700, 16, 128, "i8", 16, "f32"),
        # four users' prompts behind a shared history, grouped K/V heads
        _append("append-prompts", 4, 2001, 1003, 8, 128, "i8", 64, "bf16"),
        # one long prompt into f16 pages, the decoder model's heads
        _append("append-long-f16", 1, 7001, 0, 16, 128, "f16", 32, "f32"),
        # one decoded token of a short chat, the decoder model's heads
        _attend("attend-token", 1, 1, 500, 16, 16, 128, "i8", 16, "f32"),
        # a serving batch in decode: ragged contexts up to 4096, grouped heads
        _attend("attend-batch", 64, 1, 4096, 32, 8, 128, "i8", 16, "bf16"),
        # one decoded token on a long document
        _attend("attend-document", 1, 1, 100001, 32, 8, 128, "i8", 64, "f16"),
        # the decoder model's prompt of 500 tokens
        _attend("attend-prompt", 1, 500, 0, 16, 16, 128, "f16", 16, "f32"),
        # the next pieces of three prompts, on thousands of cached tokens
        _attend("attend-pieces", 3, 701, 6001, 32, 8, 128, "i8", 64, "bf16"),
        # a whole long prompt at once
        _attend("attend-long", 1, 8000, 0, 32, 8, 128, "i8", 128, "f16"),
        # one decoded token's alternatives
        _logprobs("logprobs-token", 1, 32000, 0, "f32", 1, 5),
        # a batch in decode with a large vocabulary and 20 alternatives
        _logprobs("logprobs-batch", 64, 128001, 63, "bf16", 1, 20),
        # the tokens of a prompt scored
        _logprobs("logprobs-prompt", 1801, 32000, 0, "f32", 1, 0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choices(["append", "attend", "logprobs"], [3, 5, 3])[0]
    if kind == "logprobs":
        vocab = _log_int(rng, 1000, 150000)
        c = _logprobs("", _log_int(rng, 1, max(1, 50_000_000 // vocab)), vocab,
                      rng.choice([0, 0, rng.randint(1, 64)]), rng.choice(list(ACTS)),
                      rng.choice([0, 1, 1, 4]), rng.choice([0, 1, 5, 20, 32]))
        if not c["given"] and not c["top"]:
            c["top"] = 1
    else:
        H, KVH, hd = rng.choice([(16, 16, 128), (32, 8, 128), (32, 8, 64), (64, 8, 64),
                                 (8, 2, 256), (16, 2, 128), (8, 8, 32), (12, 4, 96)])
        kv, act = rng.choice(["i8", "i8", "f16"]), rng.choice(list(ACTS))
        page = rng.choice([16, 32, 64, 128])
        T = 1 if rng.random() < 0.4 else _log_int(rng, 2, 4000)
        B = _log_int(rng, 1, max(1, min(64, 8000 // T)))
        ctx = rng.choice([0, _log_int(rng, 1, 200000 // B)]) if T > 1 else _log_int(rng, 1, 200000 // B)
        if kind == "append":
            c = _append("", B, T, min(ctx, 30000 // B), KVH, hd, kv, page, act)
        else:
            # at most the largest listed case's score matrix
            T = min(T, int((1_900_000_000 // (B * H)) ** 0.5))
            ctx = min(ctx, max(0, 1_900_000_000 // (B * H * T) - T))
            c = _attend("", B, T, ctx, H, KVH, hd, kv, page, act)
    c.pop("name", None)
    return c


# ---- inputs ------------------------------------------------------------------


def _ragged(case):
    """Cached and new tokens of each sequence: the longest first, down to a
    quarter of the context and half of the new tokens."""
    B, T, ctx = case["B"], case["T"], case["ctx"]
    return ([ctx - b * 3 * ctx // (4 * B) for b in range(B)],
            [T - b * T // (2 * B) for b in range(B)])


def _generator(seed):
    return torch.Generator(DEV).manual_seed(seed)


@functools.lru_cache(maxsize=8)
def _rope(n, hd):
    """[n, hd / 2, 2]: cosine and sine of position * theta^(-2 i / hd)."""
    inv = THETA ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    a = torch.arange(n, dtype=torch.float64)[:, None] * inv
    return torch.stack([a.cos(), a.sin()], -1).to(torch.float32).to(DEV)


def prepare(case, seed):
    g = _generator(seed)
    s = {"case": case}
    act = ACTS[case["act"]]
    if case["kind"] == "logprobs":
        rows, V = case["rows"], case["vocab"]
        # logits of a trained head: a broad bulk and a few likely tokens
        x = torch.randn(rows, V + case["pad"], device=DEV, generator=g) * 2.5
        likely = torch.randint(0, V, (rows, 8), device=DEV, generator=g)
        x.scatter_add_(1, likely, 8 * torch.rand(rows, 8, device=DEV, generator=g))
        s["logits"] = x.to(act)
        s["given"] = torch.randint(0, V, (rows, case["given"]), device=DEV, generator=g).int()
        if case["given"]:
            s["given"][:, 0] = likely[:, 0].int()
        s["given_lp"] = torch.empty(rows, case["given"], device=DEV)
        s["entropy"] = torch.empty(rows, device=DEV)
        s["top_id"] = torch.empty(rows, case["top"], dtype=torch.int32, device=DEV)
        s["top_lp"] = torch.empty(rows, case["top"], device=DEV)
        return s
    B, KVH, H, hd, P = (case[k] for k in ("B", "KVH", "H", "hd", "page"))
    lens, new = _ragged(case)
    held = [-(-(n + t) // P) for n, t in zip(lens, new)]
    max_pages, n_pages, N = max(held), sum(held) + 3, sum(new)
    order = torch.randperm(n_pages, device=DEV, generator=g).int()
    pages = torch.full((B, max_pages), -1, dtype=torch.int32)
    at = 0
    order = order.cpu()
    for b in range(B):
        pages[b, :held[b]] = order[at:at + held[b]]
        at += held[b]
    starts = [0]
    for t in new:
        starts.append(starts[-1] + t)
    s.update(n_pages=n_pages, max_pages=max_pages, n_rows=N, max_new=max(new),
             pages=pages.to(DEV), lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
             starts=torch.tensor(starts, dtype=torch.int32, device=DEV),
             rope=_rope(max_pages * P, hd))
    shape = (n_pages, KVH, P // 16, 16 * hd)
    if case["kv"] == "i8":
        # codes of N(0, 1) values whose page's largest is 3.6, and its scale
        for name in ("k", "v"):
            x = torch.randn(shape, device=DEV, generator=g) * (127 / 3.6)
            s[name] = x.round_().clamp_(-127, 127).to(torch.int8)
        s["scale"] = torch.exp(0.2 * torch.randn(n_pages, KVH, 2, device=DEV, generator=g)) * (3.6 / 127)
    else:
        for name in ("k", "v"):
            s[name] = torch.randn(shape, device=DEV, generator=g).half()
        s["scale"] = None
    if case["kind"] == "append":
        # the rows of one projection: keys, then values
        s["kv_new"] = torch.randn(N, 2 * KVH * hd, device=DEV, generator=g).to(act)
        # the pages that the call touches: from the start of the first one on
        first = [n - n % P for n in lens]
        rows = [n + t - f for n, t, f in zip(lens, new, first)]
        starts = [0]
        for t in rows:
            starts.append(starts[-1] + t)
        s.update(read_lens=torch.tensor(first, dtype=torch.int32, device=DEV),
                 read_starts=torch.tensor(starts, dtype=torch.int32, device=DEV),
                 read_rows=starts[-1], read_new=max(rows))
        if case["kv"] == "i8":
            s["k_out"] = torch.empty(starts[-1], KVH * hd, dtype=act, device=DEV)
            s["v_out"] = torch.empty(starts[-1], KVH * hd, dtype=act, device=DEV)
    else:
        s["q"] = torch.randn(N, H * hd, device=DEV, generator=g).to(act)
        s["out"] = torch.empty(N, H * hd, dtype=act, device=DEV)
    return s


# ---- one pass ----------------------------------------------------------------


def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"append": _own_append, "attend": _own_attend, "logprobs": _own_logprobs}[kind](s)
    return {"append": _plain_append, "attend": _plain_attend, "logprobs": _plain_logprobs}[kind](s)


def _plan(s):
    """The descriptors that a program keeps beside its cache."""
    import leafcutterllm_amd as L

    if "plan" in s:
        return L, s["plan"]
    c = s["case"]
    types = {"f32": L.TYPE_F32, "f16": L.TYPE_F16, "bf16": L.TYPE_BF16}
    if c["kind"] == "logprobs":
        n = L.logprobs_workspace(types[c["act"]], c["rows"], c["vocab"], c["given"], c["top"])
        p = {"type": types[c["act"]]}
    else:
        desc = L.KvDesc(n_head=c["H"], n_kv_head=c["KVH"], head_dim=c["hd"],
                        page_tokens=c["page"], n_pages=s["n_pages"], max_pages=s["max_pages"],
                        kv_type=L.TYPE_I8 if c["kv"] == "i8" else L.TYPE_F16,
                        act_type=types[c["act"]], rope_positions=L.ROPE_ABSOLUTE)
        p = {"desc": desc,
             "pool": L.KvPool(k=s["k"].data_ptr(), v=s["v"].data_ptr(),
                              scale=s["scale"].data_ptr() if s["scale"] is not None else None),
             "batch": L.KvBatch(n_seq=c["B"], n_rows=s["n_rows"], max_new=s["max_new"],
                                starts=s["starts"].data_ptr(), lens=s["lens"].data_ptr(),
                                pages=s["pages"].data_ptr())}
        if c["kind"] == "append":
            p["touched"] = L.KvBatch(n_seq=c["B"], n_rows=s["read_rows"], max_new=s["read_new"],
                                     starts=s["read_starts"].data_ptr(),
                                     lens=s["read_lens"].data_ptr(), pages=s["pages"].data_ptr())
        n = L.kv_attention_workspace(desc, p["batch"]) if c["kind"] == "attend" else 0
    p["ws"], p["ws_bytes"] = torch.empty(max(n, 256), dtype=torch.uint8, device=DEV), max(n, 256)
    s["plan"] = p
    return L, p


def _own_append(s):
    L, p = _plan(s)
    c = s["case"]
    st = torch.cuda.current_stream().cuda_stream
    row, kv = c["KVH"] * c["hd"], s["kv_new"]
    L.kv_append_dev(p["desc"], p["pool"], p["batch"], kv.data_ptr(), 2 * row,
                    kv.data_ptr() + row * kv.element_size(), 2 * row, s["rope"].data_ptr(), st)
    if c["kv"] == "f16":
        return s["k"], s["v"]
    L.kv_read_dev(p["desc"], p["pool"], p["touched"], s["k_out"].data_ptr(), row,
                  s["v_out"].data_ptr(), row, st)
    return s["k_out"], s["v_out"], s["scale"]


def _own_attend(s):
    L, p = _plan(s)
    c = s["case"]
    row = c["H"] * c["hd"]
    L.kv_attention_dev(p["desc"], p["pool"], p["batch"], s["q"].data_ptr(), row,
                       s["rope"].data_ptr(), c["hd"] ** -0.5, s["out"].data_ptr(), row,
                       p["ws"].data_ptr(), p["ws_bytes"], torch.cuda.current_stream().cuda_stream)
    return s["out"]


def _own_logprobs(s):
    L, p = _plan(s)
    c = s["case"]
    L.logprobs_dev(p["type"], s["logits"].data_ptr(), c["vocab"] + c["pad"], c["rows"], c["vocab"],
                   s["given"].data_ptr(), c["given"], s["given_lp"].data_ptr(),
                   s["entropy"].data_ptr(), c["top"], s["top_id"].data_ptr(),
                   s["top_lp"].data_ptr(), p["ws"].data_ptr(), p["ws_bytes"],
                   torch.cuda.current_stream().cuda_stream)
    return s["given_lp"], s["entropy"], s["top_id"], s["top_lp"]


@functools.lru_cache(maxsize=32)
def _k_places(hd, i8):
    """[16 tokens, hd] places inside a unit: for each 32 dims (8 bits: 64,
    then a last 32), four groups of dims, 16 tokens, then a group's dims."""
    r, d = torch.arange(16)[:, None], torch.arange(hd)[None, :]
    narrow = d // 32 * 512 + d % 32 // 8 * 128 + r * 8 + d % 8
    wide = d // 64 * 1024 + d % 64 // 16 * 256 + r * 16 + d % 16
    return (torch.where(d < hd // 64 * 64, wide, narrow) if i8 else narrow).to(DEV)


@functools.lru_cache(maxsize=32)
def _v_places(hd, i8):
    """[16 tokens, hd] places inside a unit: for each 32 dims (8 bits: 64, then
    a last 32), four groups of tokens, 16 dims, the 16s of dims, a group's
    tokens."""
    r, d = torch.arange(16)[:, None], torch.arange(hd)[None, :]
    t, g, e = d // 16, r // 4, r % 4
    narrow = t // 2 * 512 + g * 128 + d % 16 * 8 + t % 2 * 4 + e
    wide = t // 4 * 1024 + g * 256 + d % 16 * 16 + t % 4 * 4 + e
    return (torch.where(d < hd // 64 * 64, wide, narrow) if i8 else narrow).to(DEV)


def _rows(starts, lens, n_rows):
    """The sequence of each row and its position."""
    i = torch.arange(n_rows, device=DEV)
    b = torch.searchsorted(starts[1:].long(), i, right=True)
    return b, lens[b].long() + i - starts[b].long()


def _rotate(x, cs):
    h = x.shape[-1] // 2
    c, s = cs[..., 0], cs[..., 1]
    return torch.cat([x[..., :h] * c - x[..., h:] * s, x[..., :h] * s + x[..., h:] * c], -1)


def _plain_append(s):
    c = s["case"]
    KVH, hd, P, i8 = c["KVH"], c["hd"], c["page"], c["kv"] == "i8"
    b, pos = _rows(s["starts"], s["lens"], s["n_rows"])
    page = s["pages"][b, pos // P].long()
    # 64 bits: codes next to the border between two
    x = s["kv_new"].double().view(-1, 2, KVH, hd)
    new = {"k": _rotate(x[:, 0], s["rope"].double()[pos][:, None]), "v": x[:, 1]}
    head = torch.arange(KVH, device=DEV)[None, :, None]
    where = page[:, None, None], head, (pos % P // 16)[:, None, None]
    if not i8:
        for name, place in (("k", _k_places(hd, False)), ("v", _v_places(hd, False))):
            s[name].index_put_((*where, place[pos % 16][:, None, :]), new[name].half())
        return s["k"], s["v"]
    # each sequence's first page keeps the tokens before the call's
    seq = torch.arange(c["B"], device=DEV)
    lens = s["lens"].long()
    part = s["pages"][seq, (lens // P).clamp(max=s["max_pages"] - 1)].long()
    kept = (lens % P > 0) & (s["starts"][1:] > s["starts"][:-1])
    tok = torch.arange(P, device=DEV)
    touched = torch.zeros(s["n_pages"], 1, dtype=torch.bool, device=DEV).index_fill_(0, page, True)
    for j, (name, place) in enumerate((("k", _k_places(hd, True)), ("v", _v_places(hd, True)))):
        y = new[name]
        most = torch.zeros(s["n_pages"], KVH, dtype=torch.float64, device=DEV)
        most.index_reduce_(0, page, y.abs().amax(-1), "amax")
        before = torch.zeros(s["n_pages"], KVH, device=DEV)
        before[part] = torch.where(kept[:, None], s["scale"][part, :, j], before[part])
        scale = torch.maximum(before, (most / 127).float())
        ratio = (before.double() / scale.double())[part][:, None, :, None]
        at = (part[:, None, None, None], head[None], (tok // 16)[None, :, None, None],
              place[tok % 16][None, :, None, :])
        old = s[name][at]
        mine = kept[:, None, None, None] & (tok[None, :] < lens[:, None] % P)[:, :, None, None]
        s[name].index_put_(at, torch.where(mine, (old.double() * ratio).round().to(torch.int8), old))
        code = (y / scale.double()[page][..., None]).round().clamp(-127, 127).to(torch.int8)
        s[name].index_put_((*where, place[pos % 16][:, None, :]), code)
        s["scale"][:, :, j] = torch.where(touched, scale, s["scale"][:, :, j])
    b, pos = _rows(s["read_starts"], s["read_lens"], s["read_rows"])
    page = s["pages"][b, pos // P].long()
    out = []
    for j, (name, place) in enumerate((("k", _k_places(hd, True)), ("v", _v_places(hd, True)))):
        code = s[name][page[:, None, None], head, (pos % P // 16)[:, None, None],
                       place[pos % 16][:, None, :]]
        x = code.float() * s["scale"][page, :, j][..., None]
        out.append(x.view(-1, KVH * hd).to(ACTS[c["act"]]))
    return out[0], out[1], s["scale"]


def _plain_attend(s):
    c = s["case"]
    B, T, H, KVH, hd, P, i8 = c["B"], s["max_new"], c["H"], c["KVH"], c["hd"], c["page"], c["kv"] == "i8"
    G = H // KVH
    # dense keys and values [B, KVH, tokens, hd] of every page a sequence may hold
    pages = s["pages"].long().clamp(min=0)
    dense = []
    for j, (name, place) in enumerate((("k", _k_places(hd, i8)), ("v", _v_places(hd, i8)))):
        x = s[name][pages]                                    # [B, pages, KVH, units, 16 hd]
        x = x.index_select(-1, place.reshape(-1)).float()
        if i8:
            x = x * s["scale"][pages, :, j][..., None, None]
        x = x.view(B, -1, KVH, P // 16, 16, hd).permute(0, 2, 1, 3, 4, 5)
        dense.append(x.reshape(B, KVH, -1, hd))
    k, v = dense
    # queries in rows of [B, KVH, G, T]; those past a sequence's own repeat its last
    i = torch.arange(T, device=DEV)[None, :]
    n = (s["starts"][1:] - s["starts"][:-1]).long()[:, None]
    row = s["starts"][:-1].long()[:, None] + torch.minimum(i, n - 1)
    pos = s["lens"].long()[:, None] + torch.minimum(i, n - 1)
    q = s["q"].float().view(-1, H, hd)[row]                   # [B, T, H, hd]
    q = _rotate(q, s["rope"][pos][:, :, None])
    q = q.view(B, T, KVH, G, hd).permute(0, 2, 3, 1, 4).reshape(B, KVH, G * T, hd)
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()) * hd ** -0.5
    x = x.view(B, KVH, G, T, -1)
    seen = torch.arange(x.shape[-1], device=DEV)[None, None, :] <= pos[:, :, None]
    x = torch.where(seen[:, None, None], x, -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    o = torch.matmul(x.view(B, KVH, G * T, -1), v).view(B, KVH, G, T, hd)
    o = o / x.sum(-1, keepdim=True)
    o = o.permute(0, 3, 1, 2, 4).reshape(B * T, H * hd)
    b, pos = _rows(s["starts"], s["lens"], s["n_rows"])
    return o[b * T + pos - s["lens"].long()[b]].to(ACTS[c["act"]])


def _plain_logprobs(s):
    c = s["case"]
    x = s["logits"][:, :c["vocab"]].float()
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(-1, keepdim=True)
    lse = torch.log(z)
    entropy = (lse - (e * (x - m)).sum(-1, keepdim=True) / z)[:, 0]
    given = x.gather(1, s["given"].long()) - m - lse
    if not c["top"]:
        return given, entropy, s["top_id"], s["top_lp"]
    top, ids = torch.sort(x, dim=-1, descending=True, stable=True)
    return given, entropy, ids[:, :c["top"]].int(), top[:, :c["top"]] - m - lse


# ---- what a pass cannot do without -------------------------------------------


def work(case):
    a = 4 if case["act"] == "f32" else 2
    if case["kind"] == "logprobs":
        rows, V = case["rows"], case["vocab"]
        return {"bytes": rows * (V * a + 8 * case["given"] + 4 + 8 * case["top"]),
                "flops": 5.0 * rows * V}
    KVH, H, hd, P = case["KVH"], case["H"], case["hd"], case["page"]
    c = 1 if case["kv"] == "i8" else 2
    lens, new = _ragged(case)
    N = sum(new)
    if case["kind"] == "append":
        b = N * (2 * KVH * hd * (a + c) + 4 * hd)
        f = 6.0 * N * KVH * hd
        if c == 1:
            # the pages touched: codes and scales read back, values written
            held = sum(n % P + t for n, t in zip(lens, new))
            pages = sum(-(-(n % P + t) // P) for n, t in zip(lens, new))
            b += held * 2 * KVH * hd * (1 + a) + pages * KVH * 16
            f += 2.0 * held * KVH * hd
        return {"bytes": b, "flops": f}
    held = sum(n + t for n, t in zip(lens, new))
    pages = sum(-(-(n + t) // P) for n, t in zip(lens, new))
    seen = sum(t * n + t * (t + 1) // 2 for n, t in zip(lens, new))
    b = held * 2 * KVH * hd * c + pages * (4 + (8 * KVH if c == 1 else 0)) + 2 * N * H * hd * a
    return {"bytes": b, "flops": 4.0 * hd * H * seen}


# ---- the same in 64 bits -------------------------------------------------------


def _dense64(s, case, name, b, tokens):
    """Keys or values of a sequence's first `tokens` positions: [KVH, tokens, hd]."""
    hd, P, i8 = case["hd"], case["page"], case["kv"] == "i8"
    place = (_k_places if name == "k" else _v_places)(hd, i8)
    pages = s["pages"][b, :-(-tokens // P)].long()
    x = s[name][pages].double()
    if i8:
        x = x * s["scale"][pages, :, "kv".index(name)].double()[:, :, None, None]
    x = torch.stack([x[..., place[r]] for r in range(16)], -2)  # [pages, KVH, units, 16, hd]
    return x.transpose(0, 1).reshape(case["KVH"], -1, hd)[:, :tokens].contiguous()


def _turn64(x, cs):
    """x as complex numbers (first half, second half), times cos + i sin."""
    h = x.shape[-1] // 2
    z = torch.complex(x[..., :h], x[..., h:]) * torch.complex(cs[..., 0], cs[..., 1])
    return torch.cat([z.real, z.imag], -1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "logprobs":
        x = s["logits"][:, :case["vocab"]].double()
        given, entropy, top_lp = [], [], []
        for r in range(0, x.shape[0], 64):
            lp = torch.log_softmax(x[r:r + 64], -1)
            given.append(lp.gather(1, s["given"][r:r + 64].long()))
            entropy.append(-(lp.exp() * lp).sum(-1))
            top_lp.append(lp.topk(case["top"], -1).values if case["top"] else lp[:, :0])
        return torch.cat(given), torch.cat(entropy), None, torch.cat(top_lp)
    KVH, H, hd, P, i8 = case["KVH"], case["H"], case["hd"], case["page"], case["kv"] == "i8"
    lens, new = _ragged(case)
    rope = s["rope"].double()
    if case["kind"] == "attend":
        G, outs, at = H // KVH, [], 0
        for n, t, b in zip(lens, new, range(case["B"])):
            k, v = (_dense64(s, case, name, b, n + t) for name in "kv")
            q = _turn64(s["q"][at:at + t].double().view(t, H, hd), rope[n:n + t, None])
            o = torch.empty(t, H, hd, dtype=torch.float64, device=DEV)
            late = torch.arange(n + t, device=DEV)[None, :] > n + torch.arange(t, device=DEV)[:, None]
            for h in range(H):
                p = torch.matmul(q[:, h].contiguous(), k[h // G].T.contiguous()) / math.sqrt(hd)
                o[:, h] = torch.matmul(torch.softmax(p.masked_fill(late, -math.inf), -1), v[h // G])
            outs.append(o.view(t, H * hd))
            at += t
        return torch.cat(outs)
    # append: page by page
    row, at, ks, vs = KVH * hd, 0, [], []
    pools = {name: s[name].double() for name in "kv"}
    scale = s["scale"].double() if i8 else None
    for n, t, b in zip(lens, new, range(case["B"])):
        x = s["kv_new"][at:at + t].double()
        at += t
        y = {"k": _turn64(x[:, :row].view(t, KVH, hd), rope[n:n + t, None]),
             "v": x[:, row:].view(t, KVH, hd)}
        first = n - n % P
        for j, name in enumerate("kv"):
            place = (_k_places if name == "k" else _v_places)(hd, i8)
            held = _dense64(s, case, name, b, n)[:, first:].transpose(0, 1) if n % P else \
                torch.empty(0, KVH, hd, dtype=torch.float64, device=DEV)
            got = []
            for p0 in range(first, n + t, P):
                page = int(s["pages"][b, p0 // P])
                mine = y[name][max(p0, n) - n:p0 + P - n]     # [tokens, KVH, hd]
                if i8:
                    old = s["scale"][page, :, j].double() if p0 < n else torch.zeros_like(scale[page, :, j])
                    sc = torch.maximum(old, (mine.abs().amax((0, 2)) / 127).float().double())
                    scale[page, :, j] = sc
                    sc = sc[:, None]
                    if p0 < n:  # the codes that were there, in steps of the new scale
                        code = (held / old[:, None]).round()
                        got.append((code * (old[:, None] / sc)).round() * sc)
                    got.append((mine / sc).round() * sc)
                else:
                    for i in range(mine.shape[0]):
                        p = max(p0, n) + i
                        pools[name][page, :, p % P // 16].scatter_(
                            1, place[p % 16].expand(KVH, hd), mine[i])
            if i8:
                (ks if name == "k" else vs).append(torch.cat(got).reshape(-1, row))
    if not i8:
        return pools["k"], pools["v"]
    return torch.cat(ks), torch.cat(vs), scale
