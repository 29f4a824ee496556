// The attention of prompts over a paged cache; its instances are in
// kern_kv_prompt_*.hip, its launches in kern_kv_attn.hip.
//
// A block of W waves takes 32 W query rows of one K/V head ((token, query head
// of the group) pairs), a wave 32 of them, and goes over the context in steps
// of 64 tokens.  All waves share a step's keys and values, which the block
// brings into LDS as f16 while it computes the step before (8-bit codes are
// f16 values: the conversion is done once for 32 W rows).  A step of a wave is
//   S^T = K Q^T     [32 tokens x 32 rows] twice,
//   p = 2^(S - m),
//   O^T += V^T P^T  [32 dims x 32 rows] per 32 dims,
// on 32x32x16 matrix instructions with f32 sums.  The lane that holds row r and
// tokens 8 i + 4 g .. + 3 in S^T holds the same ones as an operand of P^T, so
// probabilities stay in registers.
//
// q is scaled by a power of two and enters as one f16 (bf16 activations) or as
// two; p enters as one, or as two where activations are f32.  An f16 is as
// exact for a large p as for a small one, so m need not be the maximum: it is
// raised, and the sums rescaled, only when some p would pass 2^14 from 2^6.
// 8-bit pages: the keys' scale is part of a score's factor.  The values' is
// part of p's exponent, relative to U, the largest of the steps so far:
// p' = 2^(S - m + 6 + log2(scale / U)), and l adds p' U / scale.
#pragma once

#include "kv_attend.h"

namespace lcmoe {

typedef float floatx16 __attribute__((ext_vector_type(16)));

// four codes to four f16: codes + 128 in the last bits of 1024 + (codes + 128)
__device__ __forceinline__ half4 codes4(uint32_t w) {
    w ^= 0x80808080u;
    const uint32_t a = __builtin_amdgcn_perm(0x64646464u, w, 0x07010700u);
    const uint32_t b = __builtin_amdgcn_perm(0x64646464u, w, 0x07030702u);
    const half4 h = __builtin_bit_cast(half4, uintx2{a, b});
    return h - half4{(_Float16)1152.0f, (_Float16)1152.0f, (_Float16)1152.0f, (_Float16)1152.0f};
}
__device__ __forceinline__ half8 cat(half4 a, half4 b) {
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
// the larger of the two lanes that hold a row (lane, lane ^ 32)
__device__ __forceinline__ float pair_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pair_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// steps that a block is worth, where blocks share rows
constexpr int kPromptLeast = 2;
// m of a row that has met no key
constexpr float kNone = -1e30f;
template <int ACT> constexpr int kQPieces = ACT == LCMOE_TYPE_BF16 ? 1 : 2;
template <int ACT> constexpr int kPPieces = ACT == LCMOE_TYPE_F32 ? 2 : 1;

// A step's keys and values between global memory and LDS.  A thread moves
// items of two chunks of a 16-token unit, its lane's: lane = unit * 16 + r.
// Keys (r: token): the two 8-dim halves of 16 dims.  Values (r: dim): tokens
// 4 g .. + 3 and 8 + 4 g .. + 3 of 2 (narrow) or 4 (wide) dims 16 apart.
template <bool I8, int NS, int W>
struct Staged {
    static constexpr int NJ = I8 ? NS / 2 : 0, NB = I8 ? NS & 1 : NS;  // wide, narrow blocks
    // items per lane set of 64: keys 4 (wide) or 2 (narrow) of 16 dims a
    // block, values 2 of the two token groups
    static constexpr int KW = 4 * NJ, VW = 2 * NJ, KN = 2 * NB, VN = 2 * NB;
    static constexpr int IT = KW + VW + KN + VN, PER = (IT + W - 1) / W;
    // a wide key item is one 16-byte chunk, a wide value item two; a narrow
    // item two chunks of 8 (8 bits) or 16 bytes
    uintx4 x[PER][2];

    __device__ __forceinline__ void load(const KvArgs &a, int wave, int lane, int page, int h,
                                         int unit) {
        const int r = lane & 15;
        const int64_t at = unit_base(a, page, h, unit);
#pragma unroll
        for (int k = 0; k < PER; k++) {
            int i = wave + k * W;
            if (i >= IT) break;
            if (I8 && i < KW) {
                x[k][0] = *reinterpret_cast<const uintx4 *>(a.k + at + (i >> 2) * 1024 + (i & 3) * 256 + r * 16);
            } else if (I8 && i < KW + VW) {
                i -= KW;
                const uint8_t *p = a.v + at + (i >> 1) * 1024 + (i & 1) * 256 + r * 16;
                x[k][0] = *reinterpret_cast<const uintx4 *>(p);
                x[k][1] = *reinterpret_cast<const uintx4 *>(p + 512);
            } else {
                i -= KW + VW;
                const bool value = i >= KN;
                if (value) i -= KN;
                const uint8_t *pool = value ? a.v : a.k;
                // keys: groups 2 s, 2 s + 1; values: g, g + 2
                const int g0 = value ? i & 1 : 2 * (i & 1), g1 = value ? g0 + 2 : g0 + 1;
                if constexpr (I8) {
                    const uint8_t *p = pool + at + NJ * 1024 + r * 8;
                    const uintx2 u = *reinterpret_cast<const uintx2 *>(p + g0 * 128);
                    const uintx2 v = *reinterpret_cast<const uintx2 *>(p + g1 * 128);
                    x[k][0] = uintx4{u[0], u[1], v[0], v[1]};
                } else {
                    const uint8_t *p = pool + 2 * at + (i >> 1) * 1024 + r * 16;
                    x[k][0] = *reinterpret_cast<const uintx4 *>(p + g0 * 256);
                    x[k][1] = *reinterpret_cast<const uintx4 *>(p + g1 * 256);
                }
            }
        }
    }

    // sk [2 tiles of 32 tokens][2 NS sets of 16 dims][2][32 tokens][8 dims]
    // sv [4 units][NS][2][32 dims][8 tokens]; there: whether the lane's page is
    // Returns whether a value is not finite (f16, and only where `edge` asks).
    __device__ __forceinline__ bool store(half8 *sk, half8 *sv, int wave, int lane, int tokens,
                                          bool there, bool edge) const {
        bool odd = false;
        const int unit = lane >> 4, r = lane & 15;
        half8 *kd = sk + (unit >> 1) * (2 * NS) * 64 + (unit & 1) * 16 + r;
        half8 *vd = sv + unit * NS * 64;
#pragma unroll
        for (int k = 0; k < PER; k++) {
            int i = wave + k * W;
            if (i >= IT) break;
            if (I8 && i < KW) {
                kd[i * 64] = cat(codes4(x[k][0][0]), codes4(x[k][0][1]));
                kd[i * 64 + 32] = cat(codes4(x[k][0][2]), codes4(x[k][0][3]));
            } else if (I8 && i < KW + VW) {
                i -= KW;
#pragma unroll
                for (int t = 0; t < 4; t++)
                    vd[(2 * (i >> 1) + (t >> 1)) * 64 + (i & 1) * 32 + (t & 1) * 16 + r] =
                        cat(codes4(x[k][0][t]), codes4(x[k][1][t]));
            } else {
                i -= KW + VW;
                const bool value = i >= KN;
                if (value) i -= KN;
                half4 c[4];
                if constexpr (I8) {
#pragma unroll
                    for (int t = 0; t < 4; t++) c[t] = codes4(x[k][0][t]);
                } else {
#pragma unroll
                    for (int t = 0; t < 4; t++)
                        c[t] = __builtin_bit_cast(half4, uintx2{x[k][t >> 1][2 * (t & 1)],
                                                                x[k][t >> 1][2 * (t & 1) + 1]});
                }
                const int b = 2 * NJ + (i >> 1);  // 32 dims
                if (!value) {
                    kd[(2 * b + (i & 1)) * 64] = cat(c[0], c[1]);
                    kd[(2 * b + (i & 1)) * 64 + 32] = cat(c[2], c[3]);
                } else {
                    const int g = i & 1;
                    if constexpr (!I8) {
                        // what is behind the last token, or not there, may be
                        // NaN: it would meet a p of zero
                        if (!there || tokens < 64) {
#pragma unroll
                            for (int t = 0; t < 4; t++)
#pragma unroll
                                for (int e = 0; e < 4; e++)
                                    if (!there || unit * 16 + 8 * (t >> 1) + 4 * g + e >= tokens)
                                        c[t][e] = (_Float16)0.0f;
                        }
                    }
                    if (!I8 && edge) {
                        const half4 z = c[0] * (_Float16)0.0f + c[1] * (_Float16)0.0f +
                                        c[2] * (_Float16)0.0f + c[3] * (_Float16)0.0f;
#pragma unroll
                        for (int e = 0; e < 4; e++) odd = odd || z[e] != z[e];
                    }
                    vd[b * 64 + g * 32 + r] = cat(c[0], c[2]);
                    vd[b * 64 + g * 32 + 16 + r] = cat(c[1], c[3]);
                }
            }
        }
        return odd;
    }
};

template <int ACT, bool I8, int NS, int W>
__global__ __launch_bounds__(64 * W, W == 8 ? 2 : 1) void k_attend_prompt(KvArgs a, AttendArgs t) {
    constexpr int NQ = kQPieces<ACT>, NP = kPPieces<ACT>, KS = 2 * NS;
    constexpr float kLog2e = 1.44269504088896340736f;
    __shared__ __attribute__((aligned(16))) half8 s_k[2][2 * KS * 64], s_v[2][4 * NS * 64];
    const int lane = threadIdx.x & 63, row = lane & 31, g = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = blockIdx.x % a.KVH, split = blockIdx.y, G = a.H / a.KVH;
    Tile x;
    if (!find_rows<64, 32 * W, kPromptLeast>(a, t, gridDim.x / a.KVH - 1 - blockIdx.x / a.KVH, x)) return;
    if (split >= x.parts) return;
    const int step0 = split * x.per, step1 = min(x.steps, (split + 1) * x.per);

    // pages: the lane's unit of the step that is being brought in
    const int32_t *table = a.pages + (int64_t)x.b * a.max_pages;
    const int ushift = a.plog - 4, last_unit = (x.n_tok - 1) >> 4;
    const auto page_of = [&](int step) {
        const int p = table[min(step * 4 + (lane >> 4), last_unit) >> ushift];
        return p < a.n_pages ? p : -1;
    };
    const auto unit_of = [&](int step) {
        return min(step * 4 + (lane >> 4), last_unit) & ((1 << ushift) - 1);
    };
    Staged<I8, NS, W> st;
    float sks = 0.0f, svs = 0.0f;  // scales of the lane's unit, of the step being brought in
    int page = page_of(step0);
    const auto bring = [&](int step) {
        st.load(a, wave, lane, max(page, 0), h, unit_of(step));
        if constexpr (I8) {
            const float *s = a.scale + ((int64_t)max(page, 0) * a.KVH + h) * 2;
            sks = s[0];
            svs = s[1];
        }
    };
    bring(step0);

    // the wave's rows
    const int r = x.r0 + 32 * wave + row, i = r / G;
    const bool valid = r < x.rows;
    const int pos = valid ? x.s.len0 + i : 0x7fffffff;
    const int r_last = min(x.r0 + 32 * wave + 31, x.rows - 1);
    const bool any = x.r0 + 32 * wave < x.rows;
    const int all_see = x.s.len0 + (x.r0 + 32 * wave) / G + 1;
    const int n_tok = any ? x.s.len0 + r_last / G + 1 : 0;
    half8 qf[NQ][KS];
    float mul;
    {
        const int half = a.hd / 2;
        const int64_t e = (int64_t)(x.s.row0 + i) * t.ldq + (int64_t)(h * G + r % G) * a.hd;
        const float *cs = t.rope + (int64_t)(a.rope_abs ? x.s.len0 + i : i) * a.hd;
        float y[KS][8], most = 0.0f, bad = 0.0f;
#pragma unroll
        for (int c = 0; c < KS; c++) {
            const int d = 16 * c + 8 * g;
            if (valid && d < a.hd) {
                load8<ACT>(t.q, e + d, t.vec, y[c]);
                if (t.rope) {
                    const bool up = d >= half;
                    const int o = up ? d - half : d;
                    float z[8];
                    load8<ACT>(t.q, e + (up ? o : d + half), t.vec, z);
                    const float *w = cs + 2 * o;
#pragma unroll
                    for (int k = 0; k < 8; k++)
                        y[c][k] = up ? z[k] * w[2 * k + 1] + y[c][k] * w[2 * k]
                                     : y[c][k] * w[2 * k] - z[k] * w[2 * k + 1];
                }
            } else {
#pragma unroll
                for (int k = 0; k < 8; k++) y[c][k] = 0.0f;
            }
#pragma unroll
            for (int k = 0; k < 8; k++) {
                most = fmaxf(most, fabsf(y[c][k]));
                bad = __builtin_fmaf(y[c][k], 0.0f, bad);  // NaN where y is not finite
            }
        }
        most = pair_max(most);
        bad = pair_sum(bad);
        // the row's largest to [2^14, 2^15): pieces are normal f16 values
        const int ex = most > 0.0f && most < INFINITY ? __builtin_amdgcn_frexp_expf(most) : 0;
        mul = __builtin_amdgcn_ldexpf(t.scale, ex - 15) * kLog2e + bad;
#pragma unroll
        for (int c = 0; c < KS; c++)
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float v = __builtin_amdgcn_ldexpf(y[c][k], 15 - ex);
                const _Float16 hi = (_Float16)v;
                qf[0][c][k] = hi;
                if constexpr (NQ == 2) qf[1][c][k] = (_Float16)(v - (float)hi);
            }
    }

    floatx16 acc[NS];
#pragma unroll
    for (int d = 0; d < NS; d++)
#pragma unroll
        for (int e = 0; e < 16; e++) acc[d][e] = 0.0f;
    // m: below every score at first; l: 2^6 sum of 2^(S - m), the lane's share
    float m = kNone, l = 0.0f, U = 0.0f;
    int buf = 0;
    // whether some row of the block does not see all of a step
    const auto edge_of = [&](int step) { return (step + 1) * 64 > x.all_see; };
    bool odd = st.store(s_k[0], s_v[0], wave, lane, x.n_tok - step0 * 64, page >= 0, edge_of(step0));
    int there = page;
    float ks_now = sks, vs_now = svs;
    page = page_of(min(step0 + 1, x.steps - 1));
    // the step's barrier; where it matters, odd becomes the block's
    const auto meet = [&](bool edge) {
        if (!I8 && edge) odd = __syncthreads_or(odd);
        else __syncthreads();
    };
    meet(edge_of(step0));
    for (int step = step0; step < step1; step++) {
        const uint64_t have = __ballot(there >= 0);
        bool missing = false;
        float ks[4], vs[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            missing = missing || !(have >> (16 * u) & 1);
            if constexpr (I8) {
                ks[u] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ks_now), 16 * u));
                vs[u] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vs_now), 16 * u));
                if (!(have >> (16 * u) & 1)) ks[u] = vs[u] = 0.0f;
            }
        }
        const bool more = step + 1 < step1;
        int next_page = 0;
        if (more) {
            bring(step + 1);
            next_page = page_of(min(step + 2, x.steps - 1));
        }
        if (step * 64 < n_tok) {
            floatx16 c[2];
#pragma unroll
            for (int tt = 0; tt < 2; tt++)
#pragma unroll
                for (int e = 0; e < 16; e++) c[tt][e] = 0.0f;
#pragma unroll
            for (int s = 0; s < KS; s++)
#pragma unroll
                for (int tt = 0; tt < 2; tt++) {
                    const half8 ka = s_k[buf][(tt * KS + s) * 64 + lane];
#pragma unroll
                    for (int p = 0; p < NQ; p++)
                        c[tt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka, qf[p][s], c[tt], 0, 0, 0);
                }
            const bool whole = !missing && (step + 1) * 64 <= all_see;
            // exponents' factors and offsets by unit; l's weights
            float f[4], off[4], weight[4];
            if constexpr (I8) {
                const float vmax = fmaxf(fmaxf(vs[0], vs[1]), fmaxf(vs[2], vs[3]));
                if (vmax > U) {
                    const float k = U / vmax;
#pragma unroll
                    for (int d = 0; d < NS; d++) acc[d] *= k;
                    U = vmax;
                }
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    // codes of a page without values are zeros, in any scale;
                    // under 2^-60 of U none of them is left in f16
                    const float w = vs[u] > 0.0f ? fmaxf(vs[u] / U, 0x1p-60f) : 1.0f;
                    f[u] = mul * ks[u];
                    off[u] = 6.0f + __builtin_amdgcn_logf(w);
                    weight[u] = 1.0f / w;
                }
            } else {
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    f[u] = mul;
                    off[u] = 6.0f;
                    weight[u] = 1.0f;
                }
            }
            // exponents S - m + off, in place; S alone while some row has no m
            const bool fresh = __ballot(m == kNone) != 0;
            float base[4], largest[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                base[u] = fresh ? 0.0f : off[u] - m;
                largest[u] = -INFINITY;
            }
#pragma unroll
            for (int tt = 0; tt < 2; tt++)
#pragma unroll
                for (int e = 0; e < 16; e++)
                    c[tt][e] = __builtin_fmaf(c[tt][e], f[2 * tt + e / 8], base[2 * tt + e / 8]);
            if (!whole) {
#pragma unroll
                for (int tt = 0; tt < 2; tt++)
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const int tok = step * 64 + 32 * tt + 8 * (e / 4) + 4 * g + e % 4;
                        if (tok > pos || !(have >> (16 * (2 * tt + e / 8)) & 1)) c[tt][e] = -INFINITY;
                    }
            }
#pragma unroll
            for (int tt = 0; tt < 2; tt++)
#pragma unroll
                for (int e = 0; e < 16; e++)
                    largest[2 * tt + e / 8] = fmaxf(largest[2 * tt + e / 8], c[tt][e]);
            const float most = fmaxf(fmaxf(largest[0], largest[1]), fmaxf(largest[2], largest[3]));
            if (fresh || __ballot(most > 14.0f)) {
                // raise m to the row's largest score, and the sums with it
                float top = m;
#pragma unroll
                for (int u = 0; u < 4; u++) top = fmaxf(top, largest[u] - base[u]);
                top = pair_max(top);
                const float keep = __builtin_amdgcn_exp2f(m - top);
                m = top;
                l *= keep;
#pragma unroll
                for (int d = 0; d < NS; d++) acc[d] *= keep;
#pragma unroll
                for (int tt = 0; tt < 2; tt++)
#pragma unroll
                    for (int e = 0; e < 16; e++)
                        c[tt][e] += (off[2 * tt + e / 8] - m) - base[2 * tt + e / 8];
            }
            // p, its pieces and its sum
            half8 pf[NP][4];
#pragma unroll
            for (int tt = 0; tt < 2; tt++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    float sum = 0.0f;
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const float p = __builtin_amdgcn_exp2f(c[tt][8 * j + e]);
                        sum += p;
                        const _Float16 hi = (_Float16)p;
                        pf[0][2 * tt + j][e] = hi;
                        if constexpr (NP == 2) pf[1][2 * tt + j][e] = (_Float16)(p - (float)hi);
                    }
                    l = __builtin_fmaf(sum, weight[2 * tt + j], l);
                }
            if (I8 || !odd || whole) {
#pragma unroll
                for (int u = 0; u < 4; u++)
#pragma unroll
                    for (int d = 0; d < NS; d++) {
                        const half8 va = s_v[buf][(u * NS + d) * 64 + lane];
#pragma unroll
                        for (int p = 0; p < NP; p++)
                            acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, pf[p][u], acc[d], 0, 0, 0);
                    }
            } else {
                // values that are not finite meet only the rows that see them,
                // whose sums they leave NaN
#pragma unroll 1
                for (int u = 0; u < 4; u++) {
                    half8 see, pu[NP];
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        const int tok = step * 64 + 16 * u + 8 * (k / 4) + 4 * g + k % 4;
                        see[k] = tok <= pos ? (_Float16)1.0f : (_Float16)0.0f;
                    }
#pragma unroll
                    for (int p = 0; p < NP; p++)
                        pu[p] = u == 0 ? pf[p][0] : u == 1 ? pf[p][1] : u == 2 ? pf[p][2] : pf[p][3];
#pragma unroll
                    for (int d = 0; d < NS; d++) {
                        half8 va = s_v[buf][(u * NS + d) * 64 + lane], is;
#pragma unroll
                        for (int k = 0; k < 8; k++) {
                            const _Float16 z = va[k] * (_Float16)0.0f;
                            is[k] = z == z ? (_Float16)0.0f : (_Float16)1.0f;
                            va[k] = z == z ? va[k] : (_Float16)0.0f;
                        }
                        floatx16 seen;
#pragma unroll
                        for (int e = 0; e < 16; e++) seen[e] = 0.0f;
                        seen = __builtin_amdgcn_mfma_f32_32x32x16_f16(is, see, seen, 0, 0, 0);
#pragma unroll
                        for (int e = 0; e < 16; e++)
                            if (seen[e] > 0.0f) acc[d][e] = NAN;
#pragma unroll
                        for (int p = 0; p < NP; p++)
                            acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, pu[p], acc[d], 0, 0, 0);
                        __builtin_amdgcn_sched_barrier(0);  // one at a time: few registers
                    }
                }
            }
        }
        if (more) {
            odd = st.store(s_k[buf ^ 1], s_v[buf ^ 1], wave, lane, x.n_tok - (step + 1) * 64, page >= 0,
                           edge_of(step + 1));
            there = page;
            ks_now = sks;
            vs_now = svs;
            page = next_page;
        }
        meet(more && edge_of(step + 1));
        buf ^= 1;
    }
    if (!valid) return;
    l = pair_sum(l);
    const int64_t orow = x.s.row0 + i;
    const int head = h * G + r % G;
    const float unit = I8 ? U : 1.0f;
    const float inv = x.parts > 1 ? unit : l == 0.0f ? 0.0f : unit / l;
    const int64_t at = (orow * a.H + head) * t.splits + split;
#pragma unroll
    for (int d = 0; d < NS; d++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int dim = 32 * d + 8 * e + 4 * g;
            const floatx4 o = floatx4{acc[d][4 * e], acc[d][4 * e + 1], acc[d][4 * e + 2],
                                      acc[d][4 * e + 3]} * inv;
            if (x.parts > 1)
                *reinterpret_cast<floatx4 *>(t.part_o + at * (32 * NS) + dim) = o;
            else if (dim < a.hd)
                store4_any(ACT, t.out, orow * t.ldo + (int64_t)head * a.hd + dim, t.vec, o);
        }
    if (x.parts > 1 && g == 0) {
        t.part_ml[2 * at] = m;
        t.part_ml[2 * at + 1] = l;
    }
}

template <int ACT>
hipError_t prompt_launch(const KvArgs &a, const AttendArgs &t, int tiles, int waves, hipStream_t st) {
    const dim3 grid((unsigned)tiles * a.KVH, t.splits);
    const auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(64 * waves), 0, st, a, t); };
    by_dims(a, [&](auto ns) {
        constexpr int NS = decltype(ns)::value;
        if constexpr (NS <= 4) {  // 2 waves or 8
            if (waves == 2) a.i8 ? go(k_attend_prompt<ACT, true, NS, 2>) : go(k_attend_prompt<ACT, false, NS, 2>);
            else a.i8 ? go(k_attend_prompt<ACT, true, NS, 8>) : go(k_attend_prompt<ACT, false, NS, 8>);
        } else {  // 4: two would hold too much of a step in registers, eight too much of q
            a.i8 ? go(k_attend_prompt<ACT, true, NS, 4>) : go(k_attend_prompt<ACT, false, NS, 4>);
        }
    });
    return waves == 2   ? attend_join<64, 64, kPromptLeast>(a, t, tiles, st)
           : waves == 4 ? attend_join<64, 128, kPromptLeast>(a, t, tiles, st)
                        : attend_join<64, 256, kPromptLeast>(a, t, tiles, st);
}

}  // namespace lcmoe
