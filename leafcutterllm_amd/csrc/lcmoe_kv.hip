// C entry points of the paged K/V cache and of the log probabilities
// (lcmoe_kv_*, lcmoe_logprobs*, include/lcmoe.h): argument checks and
// launches.  Nothing here allocates or waits, but for the host form
// lcmoe_logprobs.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "kernels.h"
#include "lcmoe_internal.h"

using namespace lcmoe;

#define HIP_TRY(expr)                                                                    \
    do {                                                                                 \
        hipError_t e_ = (expr);                                                          \
        if (e_ != hipSuccess)                                                            \
            return fail(LCMOE_ERR_HIP, "%s: %s", #expr, hipGetErrorString(e_));          \
    } while (0)

namespace {

// Launches go to the stream's device, whichever is current.
struct OnDeviceOf {
    int back = -1;
    hipError_t err = hipSuccess;
    explicit OnDeviceOf(void *stream) {
        if (!stream) return;
        int now = 0;
        hipDevice_t of = 0;
        if ((err = hipGetDevice(&now)) != hipSuccess) return;
        if ((err = hipStreamGetDevice((hipStream_t)stream, &of)) != hipSuccess) return;
        if (of != now && (err = hipSetDevice(of)) == hipSuccess) back = now;
    }
    ~OnDeviceOf() {
        if (back >= 0) (void)hipSetDevice(back);
    }
};

// the dims a head is held as: a multiple of 32, past 128 one of 64
int padded_dim(int hd) { return hd <= 128 ? (hd + 31) & ~31 : (hd + 63) & ~63; }

bool act_ok(int t) {
    return t == LCMOE_TYPE_F32 || t == LCMOE_TYPE_F16 || t == LCMOE_TYPE_BF16;
}
int act_bytes(int t) { return t == LCMOE_TYPE_F32 ? 4 : 2; }

lcmoe_status check_desc(const lcmoe_kv_desc *d) {
    if (!d) return fail(LCMOE_ERR_INVALID_ARG, "desc is NULL");
    if (d->n_head < 1 || d->n_kv_head < 1 || d->n_head % d->n_kv_head || d->n_head > 65535)
        return fail(LCMOE_ERR_INVALID_ARG,
                    "n_head=%d must be a positive multiple of n_kv_head=%d, at most 65535",
                    d->n_head, d->n_kv_head);
    if (d->head_dim < 16 || d->head_dim > 256 || d->head_dim % 16)
        return fail(LCMOE_ERR_INVALID_ARG, "head_dim=%d must be a multiple of 16 in [16, 256]",
                    d->head_dim);
    const int p = d->page_tokens;
    if (p < 16 || p > 256 || (p & (p - 1)))
        return fail(LCMOE_ERR_INVALID_ARG, "page_tokens=%d must be 16, 32, 64, 128 or 256", p);
    if (d->n_pages < 1) return fail(LCMOE_ERR_INVALID_ARG, "n_pages=%d", d->n_pages);
    if (d->max_pages < 1 || d->max_pages > (INT32_MAX - 65536) / p)
        return fail(LCMOE_ERR_INVALID_ARG, "max_pages=%d of %d tokens", d->max_pages, p);
    if (d->kv_type != LCMOE_TYPE_F16 && d->kv_type != LCMOE_TYPE_I8)
        return fail(LCMOE_ERR_UNSUPPORTED, "kv_type=%d (F16 or I8)", d->kv_type);
    if (!act_ok(d->act_type))
        return fail(LCMOE_ERR_UNSUPPORTED, "act_type=%d (F32, F16 or BF16)", d->act_type);
    if (d->rope_positions != LCMOE_ROPE_PER_CALL && d->rope_positions != LCMOE_ROPE_ABSOLUTE)
        return fail(LCMOE_ERR_INVALID_ARG, "rope_positions=%d", d->rope_positions);
    return LCMOE_OK;
}

// the batch's counts; its arrays only with `arrays`
lcmoe_status check_batch(const lcmoe_kv_batch *b, bool arrays) {
    if (!b) return fail(LCMOE_ERR_INVALID_ARG, "batch is NULL");
    if (b->n_seq < 0 || b->n_rows < 0 || b->max_new < 0 || b->n_seq > (1 << 20) ||
        b->n_rows > (1 << 30) || b->max_new > (1 << 30))
        return fail(LCMOE_ERR_INVALID_ARG, "n_seq=%d n_rows=%d max_new=%d", b->n_seq, b->n_rows,
                    b->max_new);
    if (!b->starts && arrays && (int64_t)b->n_seq * b->max_new != b->n_rows)
        return fail(LCMOE_ERR_INVALID_ARG,
                    "without starts every sequence has max_new rows: n_rows=%d, not %d * %d",
                    b->n_rows, b->n_seq, b->max_new);
    if (arrays && b->n_seq && b->n_rows && b->max_new) {
        if (!b->lens || !b->pages) return fail(LCMOE_ERR_INVALID_ARG, "lens or pages is NULL");
        if (((uintptr_t)b->starts | (uintptr_t)b->lens | (uintptr_t)b->pages) & 3)
            return fail(LCMOE_ERR_INVALID_ARG, "starts, lens and pages must be 4-byte aligned");
    }
    return LCMOE_OK;
}

// the attention counts its rows, a (token, head) each, in 31 bits
lcmoe_status check_attended(const lcmoe_kv_desc *d, const lcmoe_kv_batch *b) {
    if (((int64_t)b->n_rows + b->n_seq) * d->n_head > INT32_MAX)
        return fail(LCMOE_ERR_INVALID_ARG, "n_rows=%d (and n_seq=%d) of n_head=%d: more than 2^31",
                    b->n_rows, b->n_seq, d->n_head);
    return LCMOE_OK;
}

lcmoe_status check_pool(const lcmoe_kv_desc *d, const lcmoe_kv_pool *p) {
    if (!p || !p->k || !p->v) return fail(LCMOE_ERR_INVALID_ARG, "pool, its k or its v is NULL");
    if (((uintptr_t)p->k | (uintptr_t)p->v) & 15)
        return fail(LCMOE_ERR_INVALID_ARG, "the pool's k and v must be 16-byte aligned");
    if (d->kv_type == LCMOE_TYPE_I8 && (!p->scale || ((uintptr_t)p->scale & 7)))
        return fail(LCMOE_ERR_INVALID_ARG, "an I8 pool needs scale, 8-byte aligned");
    return LCMOE_OK;
}

// one operand of activation rows
lcmoe_status check_rows(const char *name, const void *p, int64_t ld, int heads,
                        const lcmoe_kv_desc *d) {
    if (!p) return fail(LCMOE_ERR_INVALID_ARG, "%s is NULL", name);
    if ((uintptr_t)p & (uintptr_t)(act_bytes(d->act_type) - 1))
        return fail(LCMOE_ERR_INVALID_ARG, "%s must be aligned to its elements", name);
    if (ld < (int64_t)heads * d->head_dim || ld > ((int64_t)1 << 31))
        return fail(LCMOE_ERR_INVALID_ARG, "the rows of %s are %lld apart, and hold %d * %d", name,
                    (long long)ld, heads, d->head_dim);
    return LCMOE_OK;
}

KvArgs args_of(const lcmoe_kv_desc *d, const lcmoe_kv_pool *p, const lcmoe_kv_batch *b) {
    KvArgs a{};
    if (p) {
        a.k = static_cast<uint8_t *>(p->k);
        a.v = static_cast<uint8_t *>(p->v);
        a.scale = p->scale;
    }
    a.starts = b->starts;
    a.lens = b->lens;
    a.pages = b->pages;
    a.n_seq = b->n_seq;
    a.n_rows = b->n_rows;
    a.max_new = std::min(b->max_new, b->n_rows);
    a.H = d->n_head;
    a.KVH = d->n_kv_head;
    a.hd = d->head_dim;
    a.hdp = padded_dim(d->head_dim);
    a.plog = __builtin_ctz((unsigned)d->page_tokens);
    a.n_pages = d->n_pages;
    a.max_pages = d->max_pages;
    a.rope_abs = d->rope_positions == LCMOE_ROPE_ABSOLUTE;
    a.act = d->act_type;
    a.i8 = d->kv_type == LCMOE_TYPE_I8;
    return a;
}
bool nothing(const lcmoe_kv_batch *b) { return !b->n_seq || !b->n_rows || !b->max_new; }

lcmoe_status check_rope(const float *rope) {
    if ((uintptr_t)rope & 7) return fail(LCMOE_ERR_INVALID_ARG, "rope must be 8-byte aligned");
    return LCMOE_OK;
}

lcmoe_status check_logprobs(int32_t type, int64_t ld, int32_t rows, int32_t vocab, int32_t n_given,
                            int32_t n_top) {
    if (!act_ok(type)) return fail(LCMOE_ERR_UNSUPPORTED, "type=%d (F32, F16 or BF16)", type);
    if (rows < 0 || vocab < 1 || vocab > (1 << 30) || ld < vocab || ld > ((int64_t)1 << 40))
        return fail(LCMOE_ERR_INVALID_ARG, "n_rows=%d vocab=%d ld=%lld", rows, vocab, (long long)ld);
    if (n_given < 0 || n_given > 65536) return fail(LCMOE_ERR_INVALID_ARG, "n_given=%d outside [0, 65536]", n_given);
    if (n_top < 0 || n_top > LCMOE_LOGPROBS_TOP)
        return fail(LCMOE_ERR_INVALID_ARG, "n_top=%d outside [0, %d]", n_top, LCMOE_LOGPROBS_TOP);
    return LCMOE_OK;
}

}  // namespace

extern "C" lcmoe_status lcmoe_kv_sizes(const lcmoe_kv_desc *desc, size_t *pool_bytes,
                                       size_t *scale_bytes) {
    clear_error();
    if (lcmoe_status s = check_desc(desc)) return s;
    const size_t per_page = (size_t)desc->n_kv_head * desc->page_tokens *
                            (size_t)padded_dim(desc->head_dim);
    const bool i8 = desc->kv_type == LCMOE_TYPE_I8;
    if (pool_bytes) *pool_bytes = per_page * (size_t)desc->n_pages * (i8 ? 1 : 2);
    if (scale_bytes) *scale_bytes = i8 ? 8 * (size_t)desc->n_pages * desc->n_kv_head : 0;
    return LCMOE_OK;
}

extern "C" lcmoe_status lcmoe_kv_append_dev(const lcmoe_kv_desc *desc, const lcmoe_kv_pool *pool,
                                            const lcmoe_kv_batch *batch, const void *k_dev,
                                            int64_t ld_k, const void *v_dev, int64_t ld_v,
                                            const float *rope_dev, void *stream) {
    clear_error();
    if (lcmoe_status s = check_desc(desc)) return s;
    if (lcmoe_status s = check_batch(batch, true)) return s;
    if (nothing(batch)) return LCMOE_OK;
    if (lcmoe_status s = check_pool(desc, pool)) return s;
    if (lcmoe_status s = check_rows("k", k_dev, ld_k, desc->n_kv_head, desc)) return s;
    if (lcmoe_status s = check_rows("v", v_dev, ld_v, desc->n_kv_head, desc)) return s;
    if (lcmoe_status s = check_rope(rope_dev)) return s;
    OnDeviceOf on(stream);
    HIP_TRY(on.err);
    HIP_TRY(launch_kv_append(args_of(desc, pool, batch), k_dev, ld_k, v_dev, ld_v, rope_dev,
                             (hipStream_t)stream));
    return LCMOE_OK;
}

extern "C" lcmoe_status lcmoe_kv_read_dev(const lcmoe_kv_desc *desc, const lcmoe_kv_pool *pool,
                                          const lcmoe_kv_batch *batch, void *k_dev, int64_t ld_k,
                                          void *v_dev, int64_t ld_v, void *stream) {
    clear_error();
    if (lcmoe_status s = check_desc(desc)) return s;
    if (lcmoe_status s = check_batch(batch, true)) return s;
    if (nothing(batch)) return LCMOE_OK;
    if (lcmoe_status s = check_pool(desc, pool)) return s;
    if (lcmoe_status s = check_rows("k", k_dev, ld_k, desc->n_kv_head, desc)) return s;
    if (lcmoe_status s = check_rows("v", v_dev, ld_v, desc->n_kv_head, desc)) return s;
    OnDeviceOf on(stream);
    HIP_TRY(on.err);
    HIP_TRY(launch_kv_read(args_of(desc, pool, batch), k_dev, ld_k, v_dev, ld_v,
                           (hipStream_t)stream));
    return LCMOE_OK;
}

extern "C" lcmoe_status lcmoe_kv_attention_workspace(const lcmoe_kv_desc *desc,
                                                     const lcmoe_kv_batch *batch, size_t *bytes) {
    clear_error();
    if (!bytes) return fail(LCMOE_ERR_INVALID_ARG, "bytes is NULL");
    if (lcmoe_status s = check_desc(desc)) return s;
    if (lcmoe_status s = check_batch(batch, false)) return s;
    if (lcmoe_status s = check_attended(desc, batch)) return s;
    *bytes = nothing(batch) ? 0 : 4 * (size_t)kv_attention_floats(args_of(desc, nullptr, batch));
    return LCMOE_OK;
}

extern "C" lcmoe_status lcmoe_kv_attention_dev(const lcmoe_kv_desc *desc, const lcmoe_kv_pool *pool,
                                               const lcmoe_kv_batch *batch, const void *q_dev,
                                               int64_t ld_q, const float *rope_dev, float scale,
                                               void *out_dev, int64_t ld_out, void *workspace,
                                               size_t workspace_bytes, void *stream) {
    clear_error();
    if (lcmoe_status s = check_desc(desc)) return s;
    if (lcmoe_status s = check_batch(batch, true)) return s;
    if (lcmoe_status s = check_attended(desc, batch)) return s;
    if (!(scale > 0.0f) || !std::isfinite(scale))
        return fail(LCMOE_ERR_INVALID_ARG, "scale must be finite and > 0");
    if (nothing(batch)) return LCMOE_OK;
    if (lcmoe_status s = check_pool(desc, pool)) return s;
    if (lcmoe_status s = check_rows("q", q_dev, ld_q, desc->n_head, desc)) return s;
    if (lcmoe_status s = check_rows("out", out_dev, ld_out, desc->n_head, desc)) return s;
    if (lcmoe_status s = check_rope(rope_dev)) return s;
    const KvArgs a = args_of(desc, pool, batch);
    const size_t need = 4 * (size_t)kv_attention_floats(a);
    if (need && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need))
        return fail(LCMOE_ERR_INVALID_ARG, "needs a 16-byte aligned workspace of %zu bytes, got %zu",
                    need, workspace ? workspace_bytes : 0);
    OnDeviceOf on(stream);
    HIP_TRY(on.err);
    HIP_TRY(launch_kv_attention(a, q_dev, ld_q, rope_dev, scale, out_dev, ld_out,
                                static_cast<float *>(workspace), (hipStream_t)stream));
    return LCMOE_OK;
}

extern "C" lcmoe_status lcmoe_logprobs_workspace(int32_t type, int32_t n_rows, int32_t vocab,
                                                 int32_t n_given, int32_t n_top, size_t *bytes) {
    clear_error();
    if (!bytes) return fail(LCMOE_ERR_INVALID_ARG, "bytes is NULL");
    if (lcmoe_status s = check_logprobs(type, vocab, n_rows, vocab, n_given, n_top)) return s;
    *bytes = n_rows ? (size_t)logprobs_bytes(type, n_rows, vocab, n_top) : 0;
    return LCMOE_OK;
}

extern "C" lcmoe_status lcmoe_logprobs_dev(int32_t type, const void *logits_dev, int64_t ld,
                                           int32_t n_rows, int32_t vocab, const int32_t *given_dev,
                                           int32_t n_given, float *given_lp_dev, float *entropy_dev,
                                           int32_t n_top, int32_t *top_id_dev, float *top_lp_dev,
                                           void *workspace, size_t workspace_bytes, void *stream) {
    clear_error();
    if (lcmoe_status s = check_logprobs(type, ld, n_rows, vocab, n_given, n_top)) return s;
    if (!n_rows || (!n_given && !entropy_dev && !n_top)) return LCMOE_OK;
    if (!logits_dev || (n_given && (!given_dev || !given_lp_dev)) ||
        (n_top && (!top_id_dev || !top_lp_dev)))
        return fail(LCMOE_ERR_INVALID_ARG, "logits, given or a result is NULL");
    if (((uintptr_t)logits_dev & (uintptr_t)(act_bytes(type) - 1)) ||
        (((uintptr_t)given_dev | (uintptr_t)given_lp_dev | (uintptr_t)entropy_dev |
          (uintptr_t)top_id_dev | (uintptr_t)top_lp_dev) & 3))
        return fail(LCMOE_ERR_INVALID_ARG, "logits, given and the results must be aligned to their elements");
    const size_t need = (size_t)logprobs_bytes(type, n_rows, vocab, n_top);
    if (need && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need))
        return fail(LCMOE_ERR_INVALID_ARG, "needs a 16-byte aligned workspace of %zu bytes, got %zu",
                    need, workspace ? workspace_bytes : 0);
    OnDeviceOf on(stream);
    HIP_TRY(on.err);
    HIP_TRY(launch_logprobs(type, logits_dev, ld, n_rows, vocab, given_dev, n_given, given_lp_dev,
                            entropy_dev, n_top, top_id_dev, top_lp_dev, workspace,
                            (hipStream_t)stream));
    return LCMOE_OK;
}

extern "C" lcmoe_status lcmoe_logprobs(int32_t type, const void *logits, int64_t ld, int32_t n_rows,
                                       int32_t vocab, const int32_t *given, int32_t n_given,
                                       float *given_lp, float *entropy, int32_t n_top,
                                       int32_t *top_id, float *top_lp) {
    clear_error();
    if (lcmoe_status s = check_logprobs(type, ld, n_rows, vocab, n_given, n_top)) return s;
    if (!n_rows || (!n_given && !entropy && !n_top)) return LCMOE_OK;
    if (!logits || (n_given && (!given || !given_lp)) || (n_top && (!top_id || !top_lp)))
        return fail(LCMOE_ERR_INVALID_ARG, "logits, given or a result is NULL");
    const size_t R = (size_t)n_rows;
    // the last row ends at its vocabulary
    const size_t xb = ((R - 1) * (size_t)ld + vocab) * act_bytes(type);
    const size_t gb = 4 * R * n_given, tb = 4 * R * n_top;
    const size_t wb = (size_t)logprobs_bytes(type, n_rows, vocab, n_top);
    const auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    uint8_t *p = nullptr;
    hipError_t e = hipMalloc(&p, up(xb) + 2 * up(gb) + up(4 * R) + 2 * up(tb) + up(wb));
    if (e == hipErrorOutOfMemory) {
        (void)hipGetLastError();
        return fail(LCMOE_ERR_OUT_OF_MEMORY, "logprobs: %s", hipGetErrorString(e));
    }
    uint8_t *dg = p + up(xb), *dl = dg + up(gb), *de = dl + up(gb), *di = de + up(4 * R),
            *dt = di + up(tb), *dw = dt + up(tb);
    if (e == hipSuccess) e = hipMemcpy(p, logits, xb, hipMemcpyHostToDevice);
    if (e == hipSuccess && gb) e = hipMemcpy(dg, given, gb, hipMemcpyHostToDevice);
    if (e == hipSuccess)
        e = launch_logprobs(type, p, ld, n_rows, vocab, (const int32_t *)dg, n_given, (float *)dl,
                            (float *)de, n_top, (int32_t *)di, (float *)dt, dw, nullptr);
    if (e == hipSuccess && gb) e = hipMemcpy(given_lp, dl, gb, hipMemcpyDeviceToHost);
    if (e == hipSuccess && entropy) e = hipMemcpy(entropy, de, 4 * R, hipMemcpyDeviceToHost);
    if (e == hipSuccess && tb) e = hipMemcpy(top_id, di, tb, hipMemcpyDeviceToHost);
    if (e == hipSuccess && tb) e = hipMemcpy(top_lp, dt, tb, hipMemcpyDeviceToHost);
    if (p) (void)hipFree(p);
    if (e != hipSuccess) return fail(LCMOE_ERR_HIP, "logprobs: %s", hipGetErrorString(e));
    return LCMOE_OK;
}
