// The attention of prompts over a paged cache; its instances are in
// kern_kv_prompt_*.hip, its launches in kern_kv_attn.hip.
//
// A block takes 32 WR query rows of one K/V head ((token, query head of the
// group) pairs), a wave 32 of them, and goes over the context in steps of 64
// tokens.  All waves share a step's keys and values, which the block brings into
// LDS while it computes the step before.  8-bit codes are f16 values: values,
// and keys but for f16 activations, become f16 on the way, once for all rows.
// A step of a wave is
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
// 8-bit pages and f16 activations: two f16 products would be S^T; two integer
// products (32x32x32, twice the rate) of q's two signed 8-bit pieces with the
// codes themselves take half of that and half of the LDS (8000 tokens, 32 heads
// of 128: 632 us against 758; 701 tokens behind 6001, three times: 240 against
// 276).  For bf16 one f16 product is as fast, and needs no conversion of sums
// (612 against 634, 226 against 238); for f32 it would be three integer products
// and sums for each (919 against 942, 350 against 346, and 500 tokens of 16
// heads 25.9 against 18.4).
// 8-bit pages: the keys' scale is part of a score's factor.  The values' is
// part of p's exponent, relative to U, the largest of the steps so far:
// p' = 2^(S - m + 6 + log2(scale / U)), and l adds p' U / scale.
#pragma once

#include "kv_attend.h"

namespace lcmoe {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef int32_t intx16 __attribute__((ext_vector_type(16)));

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

// groups of 32 rows of a block of many, and shares of the context of one of 64
// rows: as many as the registers of a head allow
template <int NS> constexpr int kManyRows = NS <= 4 ? 8 : 4;
template <int NS> constexpr int kShares = NS <= 4 ? 4 : 2;
// steps that a block is worth, where blocks share rows
template <int WT> constexpr int kPromptLeast = 2 * WT;
// m of a row that has met no key
constexpr float kNone = -1e30f;
template <int ACT> constexpr int kQPieces = ACT == LCMOE_TYPE_BF16 ? 1 : 2;
// whether the keys' codes enter as they are
template <int ACT, bool I8> constexpr bool kCodes = I8 && ACT == LCMOE_TYPE_F16;
template <int ACT> constexpr int kPPieces = ACT == LCMOE_TYPE_F32 ? 2 : 1;

// What a load has brought, copied here: the compiler would copy it to the next
// turn's register at the end of the loop, and wait for the load there.
template <class T>
__device__ __forceinline__ T arrived(T x) {
    T y;
    asm volatile("v_mov_b32 %0, %1" : "=v"(y) : "v"(x));
    return y;
}

// A step's keys and values between global memory and LDS.  A lane moves items
// of two chunks of its 16-token unit: lane = unit * 16 + r.  Keys (r: token):
// two neighbouring groups of dims, so that an item is 32 (wide) or 16 (narrow)
// dims.  Values (r: dim): token groups g and g + 2, of 4 (wide) or 2 (narrow)
// dims 16 apart.  A wave's items are known by its number alone, and every one
// is the same two loads, so that nothing waits for a load but its store.
template <bool I8, bool CODES, int NS, int W>
struct Staged {
    static constexpr int NJ = I8 ? NS / 2 : 0, NB = I8 ? NS & 1 : NS;  // wide, narrow blocks
    // items: of each block two of keys, then two of values
    static constexpr int WI = 4 * NJ, NI = 4 * NB;
    static constexpr int PW = (WI + W - 1) / W, PN = (NI + W - 1) / W;
    uintx4 x[PW ? PW : 1][2], y[PN ? PN : 1][2];  // narrow 8-bit chunks: 8 bytes each, in y[.][0]

    __device__ __forceinline__ void load(const KvArgs &a, int wave, int lane, int page, int h,
                                         int unit) {
        const int r = lane & 15;
        const int64_t at = unit_base(a, page, h, unit) * (I8 ? 1 : 2);
#pragma unroll
        for (int k = 0; k < PW; k++) {
            const int i = min(wave + k * W, WI - 1);
            const bool value = i >= 2 * NJ;
            const int j = value ? i - 2 * NJ : i;
            const uint8_t *p = (value ? a.v : a.k) + at + (j >> 1) * 1024 + r * 16;
            x[k][0] = *reinterpret_cast<const uintx4 *>(p + (value ? 256 : 512) * (j & 1));
            x[k][1] = *reinterpret_cast<const uintx4 *>(p + (value ? 256 : 512) * (j & 1) + (value ? 512 : 256));
        }
        constexpr int C = I8 ? 8 : 16;  // bytes of a chunk
#pragma unroll
        for (int k = 0; k < PN; k++) {
            const int i = min(wave + k * W, NI - 1);
            const bool value = i >= 2 * NB;
            const int j = value ? i - 2 * NB : i;
            const uint8_t *p = (value ? a.v : a.k) + at + NJ * 1024 + (j >> 1) * 64 * C + r * C +
                               (value ? 16 : 32) * C * (j & 1);
            const int next = (value ? 32 : 16) * C;
            if constexpr (I8) {
                const uintx2 u = *reinterpret_cast<const uintx2 *>(p);
                const uintx2 v = *reinterpret_cast<const uintx2 *>(p + next);
                y[k][0] = uintx4{u[0], u[1], v[0], v[1]};
            } else {
                y[k][0] = *reinterpret_cast<const uintx4 *>(p);
                y[k][1] = *reinterpret_cast<const uintx4 *>(p + next);
            }
        }
    }

    // sk [2 tiles of 32 tokens][sets of 32 (codes) or 16 (f16) dims][2][32
    // tokens][16 bytes]; sv [4 units][NS][2][32 dims][8 tokens]; there: whether
    // the lane's page is.  f16, where `edge` asks: a value that is not finite is
    // stored as zero, and its token's bit set in bad[dim]; returns whether there
    // is one.
    __device__ __forceinline__ bool store(uintx4 *sk, half8 *sv, int wave, int lane, int tokens,
                                          bool there, bool edge, unsigned long long *bad) const {
        bool odd = false;
        const int unit = lane >> 4, r = lane & 15;
        uintx4 *kd = sk + (unit >> 1) * (CODES ? NS : 2 * NS) * 64 + (unit & 1) * 16 + r;
        half8 *vd = sv + unit * NS * 64 + r;
#pragma unroll
        for (int k = 0; k < PW; k++) {
            const int i = wave + k * W, j = i >= 2 * NJ ? i - 2 * NJ : i;
            if (i < 2 * NJ) {  // dims 64 (j / 2) + 32 (j % 2), 16 in each of x
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    if constexpr (CODES) {
                        kd[j * 64 + c * 32] = x[k][c];
                    } else {
#pragma unroll
                        for (int g = 0; g < 2; g++)
                            kd[(2 * j + c) * 64 + g * 32] = __builtin_bit_cast(
                                uintx4, cat(codes4(x[k][c][2 * g]), codes4(x[k][c][2 * g + 1])));
                    }
                }
            } else if (i < WI) {
#pragma unroll
                for (int t = 0; t < 4; t++)
                    vd[(2 * (j >> 1) + (t >> 1)) * 64 + (j & 1) * 32 + (t & 1) * 16] =
                        cat(codes4(x[k][0][t]), codes4(x[k][1][t]));
            }
        }
#pragma unroll
        for (int k = 0; k < PN; k++) {
            const int i = wave + k * W;
            if (i >= NI) break;
            if (CODES && i < 2 * NB) {
                kd[2 * NJ * 64 + i * 32] = y[k][0];
                continue;
            }
            half4 c[4];  // chunk 0, chunk 1: of 8 dims, or of 2 dims by 4 tokens
#pragma unroll
            for (int t = 0; t < 4; t++)
                c[t] = I8 ? codes4(y[k][0][t])
                          : __builtin_bit_cast(half4, uintx2{y[k][t >> 1][2 * (t & 1)],
                                                             y[k][t >> 1][2 * (t & 1) + 1]});
            if (i < 2 * NB) {
                kd[(4 * NJ + i) * 64] = __builtin_bit_cast(uintx4, cat(c[0], c[1]));
                kd[(4 * NJ + i) * 64 + 32] = __builtin_bit_cast(uintx4, cat(c[2], c[3]));
            } else {
                const int j = i - 2 * NB, g = j & 1, b = 2 * NJ + (j >> 1);
                if constexpr (!I8) {
                    // what is behind the last token, or not there, may be NaN:
                    // it would meet a p of zero
                    if (!there || tokens < 64) {
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const int n = there ? min(max(tokens - unit * 16 - 8 * h - 4 * g, 0), 4) : 0;
                            const uint64_t keep = n == 4 ? ~0ull : (1ull << 16 * n) - 1;
#pragma unroll
                            for (int t = 2 * h; t < 2 * h + 2; t++)
                                c[t] = __builtin_bit_cast(half4, __builtin_bit_cast(uint64_t, c[t]) & keep);
                        }
                    }
                    const half4 z = (c[0] + c[1] + c[2] + c[3]) * (_Float16)0.0f;
                    if (edge && __builtin_expect(
                                    __ballot(z[0] + z[1] + z[2] + z[3] != (_Float16)0.0f) != 0, 0)) {
#pragma unroll
                        for (int t = 0; t < 4; t++) {
                            unsigned long long bits = 0;
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const _Float16 z = c[t][e] * (_Float16)0.0f;
                                if (z == z) continue;
                                c[t][e] = (_Float16)0.0f;
                                bits |= 1ull << (unit * 16 + 8 * (t >> 1) + 4 * g + e);
                            }
                            if (bits) {
                                atomicOr(&bad[32 * b + 16 * (t & 1) + r], bits);
                                odd = true;
                            }
                        }
                    }
                }
                vd[b * 64 + g * 32] = cat(c[0], c[2]);
                vd[b * 64 + g * 32 + 16] = cat(c[1], c[3]);
            }
        }
        return odd;
    }
};

// The order of the instructions around it: LDS reads run four operands ahead
// of the `per` matrix instructions that take one.
template <int READS, int PER>
__device__ __forceinline__ void read_ahead() {
    constexpr int A = READS < 4 ? READS : 4;
    __builtin_amdgcn_sched_group_barrier(0x100, A, 0);
#pragma unroll
    for (int i = 0; i < READS; i++) {
        __builtin_amdgcn_sched_group_barrier(0x008, PER, 0);
        if (i + A < READS) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
}

// WR WT waves: WR groups of 32 rows, WT shares of the context, which take the
// block's steps in turn, each with buffers of its own, and add up at the end.
// WT = 1: two buffers, so that a step is brought in beside the one before.
template <int ACT, bool I8, int NS, int WR, int WT>
__global__ __launch_bounds__(64 * WR * WT, NS <= 4 ? 2 : 1) void k_attend_prompt(KvArgs a, AttendArgs t) {
    constexpr bool CODES = kCodes<ACT, I8>;
    constexpr int NQ = kQPieces<ACT>, NP = kPPieces<ACT>, KS = CODES ? NS : 2 * NS, M = 32 * WR;
    // f16 pages, q's last piece: where registers would not hold it, it stays in
    // LDS, which has the bandwidth to read it again each step.  Heads of 128 (and
    // 96) dims: 8000 tokens of 32 heads 854 us against 1156, bf16 activations 676
    // against 716, 500 tokens of 16 heads 18.3 against 23.0.  Past 192 dims, in
    // the room of the second buffer: 4000 tokens of 16 heads of 256 279 us against
    // 934.  Smaller heads have the registers; blocks of 64 rows of larger ones
    // have not the LDS.
    constexpr bool LOW = !I8 && (WT == 1 ? NS == 3 || NS == 4 || NS == 8 : NS == 4);
    constexpr bool TWICE = WT == 1 && !(LOW && NS == 8);
    constexpr int SLOTS = TWICE ? 4 : 2;
    constexpr int KB = 2 * KS * 64, VB = 4 * NS * 64, BUFS = TWICE ? 2 : WT;
    constexpr int QB = WR * NQ * KS * 64, LB = LOW ? WR * KS * 64 : 0, SB = BUFS * (KB + VB) + LB;
    __shared__ __attribute__((aligned(16))) half8 s_kv[SB > QB ? SB : QB];
    __shared__ float s_mul[M];
    // f16 pages: of a step that not every row of the block sees, the tokens
    // whose values are not finite, by dim; by turn, and whether there are any
    __shared__ unsigned long long s_bad[I8 ? 1 : WT * SLOTS][I8 ? 1 : 32 * NS];
    __shared__ int s_odd[WT][SLOTS];
    uintx4 *const s_k = reinterpret_cast<uintx4 *>(s_kv);
    half8 *const s_v = s_kv + BUFS * KB;
    const int lane = threadIdx.x & 63, row = lane & 31, g = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave % WR, wt = wave / WR;
    const int h = blockIdx.x % a.KVH, split = blockIdx.y, G = a.H / a.KVH;
    Tile x;
    if (!find_rows<64, M, kPromptLeast<WT>>(a, t, gridDim.x / a.KVH - 1 - blockIdx.x / a.KVH, x)) return;
    if (split >= x.parts) return;
    const int step0 = split * x.per + wt, step1 = min(x.steps, (split + 1) * x.per);
    const int turns = (step1 - split * x.per + WT - 1) / WT;

    // pages: the lane's unit of the step that is being brought in
    const int32_t *table = a.pages + (int64_t)x.b * a.max_pages;
    const int ushift = a.plog - 4, last_unit = (x.n_tok - 1) >> 4;
    const auto page_of = [&](int step) {
        return table[min(step * 4 + (lane >> 4), last_unit) >> ushift];
    };
    const auto is_there = [&](int p) { return p >= 0 && p < a.n_pages; };
    Staged<I8, CODES, NS, WR> st;
    float sks = 0.0f, svs = 0.0f;  // scales of the lane's unit, of the step being brought in
    int page = page_of(step0);
    const auto bring = [&](int step) {
        const int p = is_there(page) ? page : 0;
        st.load(a, wr, lane, p, h, min(step * 4 + (lane >> 4), last_unit) & ((1 << ushift) - 1));
        if constexpr (I8) {
            const float *s = a.scale + ((int64_t)p * a.KVH + h) * 2;
            sks = s[0];
            svs = s[1];
        }
    };
    bring(step0);
    int page_ahead = page_of(step0 + WT);

    // the wave's rows
    const int first = x.r0 + 32 * wr, r = first + row, i = r / G;
    const bool valid = r < x.rows;
    const int pos = valid ? x.s.len0 + i : 0x7fffffff;
    const int all_see = x.s.len0 + first / G + 1;
    const int n_tok = first < x.rows ? x.s.len0 + min(first + 31, x.rows - 1) / G + 1 : 0;
    if constexpr (!I8) {
#pragma unroll 1
        for (int k = threadIdx.x; k < WT * SLOTS * 32 * NS; k += 64 * WR * WT) (&s_bad[0][0])[k] = 0;
        if (threadIdx.x < SLOTS * WT) (&s_odd[0][0])[threadIdx.x] = 0;
    }
    // its operands, through LDS: [group of rows][piece][set of dims][lane]
    uintx4 *const s_q = s_k;
    stage_q<NS, M, 64 * WR * WT>(a, t, x, h,
        [&](int64_t e, float (&y)[8]) { load_n<ACT>(t.q, e, y); },
        [&](int r, int c, const float (&y)[8], float most) {
            if constexpr (CODES) {
                uint32_t o0[NQ], o1[NQ];
                Ops<true, NQ, NS>::pieces(&y[0], most, o0);
                Ops<true, NQ, NS>::pieces(&y[4], most, o1);
#pragma unroll
                for (int p = 0; p < NQ; p++)
                    reinterpret_cast<uintx2 *>(
                        s_q + (((r >> 5) * NQ + p) * KS + (c >> 2)) * 64 + (c >> 1 & 1) * 32 + (r & 31))[c & 1] =
                        uintx2{o0[p], o1[p]};
            } else {
                half8 o[NQ];
                half_pieces<NQ>(y, exponent_of(most), o);
#pragma unroll
                for (int p = 0; p < NQ; p++)
                    s_q[(((r >> 5) * NQ + p) * KS + (c >> 1)) * 64 + (c & 1) * 32 + (r & 31)] =
                        __builtin_bit_cast(uintx4, o[p]);
            }
        },
        [&](int r, float most, float bad) {
            s_mul[r] = Ops<CODES, NQ, NS>::factor(most, t.scale) + bad;
        });
    __syncthreads();
    uintx4 qf[NQ][KS];
#pragma unroll
    for (int p = 0; p < NQ; p++)
#pragma unroll
        for (int c = 0; c < KS; c++) qf[p][c] = s_q[((wr * NQ + p) * KS + c) * 64 + lane];
    const float mul = s_mul[32 * wr + row];
    __syncthreads();  // the buffers are the steps' from here on
    uintx4 *const s_low = s_k + BUFS * (KB + VB) + wr * KS * 64 + lane;
    if (LOW && wt == 0)
#pragma unroll
        for (int c = 0; c < KS; c++) s_low[c * 64] = qf[NQ - 1][c];

    floatx16 acc[NS];
#pragma unroll
    for (int d = 0; d < NS; d++)
#pragma unroll
        for (int e = 0; e < 16; e++) acc[d][e] = 0.0f;
    // m: below every score at first; l: 2^6 sum of 2^(S - m), the lane's share
    float m = kNone, l = 0.0f, U = 0.0f, log_U = 0.0f;
    int there = page;
    float ks_now = sks, vs_now = svs;
    // whether some row of the block does not see all of a step
    const auto edge_of = [&](int step) { return (step + 1) * 64 > x.all_see; };
    const auto store = [&](int step, int n, int buf) {
        unsigned long long *const bad = s_bad[I8 ? 0 : wt * SLOTS + n % SLOTS];
        const bool odd = st.store(s_k + buf * KB, s_v + buf * VB, wr, lane, x.n_tok - step * 64,
                                  is_there(page), edge_of(step), bad);
        if constexpr (!I8) {
            if (odd) s_odd[wt][n % SLOTS] = 1;
            // of the next turn, or with two buffers the one after: its last
            // reader passed a barrier ago
            constexpr int AHEAD = SLOTS / 2;
            if (edge_of(step + AHEAD * WT)) {
                if (wr == 0 && lane == 0) s_odd[wt][(n + AHEAD) % SLOTS] = 0;
                for (int k = wr * 64 + lane; k < 32 * NS; k += 64 * WR)
                    s_bad[wt * SLOTS + (n + AHEAD) % SLOTS][k] = 0;
            }
        }
    };
    // what has arrived becomes the step's, and the next one is sent for; past
    // the last it is again: a branch would make the loads' registers wait
    const auto send = [&](int step) {
        there = page;
        if constexpr (I8) {
            ks_now = arrived(sks);
            vs_now = arrived(svs);
        }
        page = arrived(page_ahead);
        bring(step);
        page_ahead = page_of(step + WT);
    };
    if constexpr (TWICE) {
        store(step0, 0, 0);
        __syncthreads();
        send(step0 + 1);
    }
    for (int n = 0; n < turns; n++) {
        const int step = step0 + n * WT, buf = TWICE ? n & 1 : wt;
        if constexpr (!TWICE) {
            store(step, n, buf);
            __syncthreads();
            send(step + WT);
        }
        const uint64_t have = __ballot(is_there(there));
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
        if (step < step1 && step * 64 < n_tok) {
            const bool whole = !missing && (step + 1) * 64 <= all_see;
            const uintx4 *const kp = s_k + buf * KB + lane;
            const half8 *const vp = s_v + buf * VB + lane;
            floatx16 c[2];
            // a product on the same sums waits for the one before: turn by turn
            if constexpr (CODES) {
#pragma unroll
                for (int tt = 0; tt < 2; tt++) {
                    intx16 n[NQ];
#pragma unroll
                    for (int p = 0; p < NQ; p++)
#pragma unroll
                        for (int e = 0; e < 16; e++) n[p][e] = 0;
#pragma unroll
                    for (int s = 0; s < KS; s++) {
                        const intx4 ka = __builtin_bit_cast(intx4, kp[(tt * KS + s) * 64]);
#pragma unroll
                        for (int p = 0; p < NQ; p++)
                            n[p] = __builtin_amdgcn_mfma_i32_32x32x32_i8(
                                ka, __builtin_bit_cast(intx4, qf[p][s]), n[p], 0, 0, 0);
                    }
                    // at most 127 (127 256) 256 < 2^31
#pragma unroll
                    for (int e = 0; e < 16; e++) c[tt][e] = (float)(n[0][e] * 256 + n[1][e]);
                }
            } else {
#pragma unroll
                for (int tt = 0; tt < 2; tt++)
#pragma unroll
                    for (int e = 0; e < 16; e++) c[tt][e] = 0.0f;
#pragma unroll
                for (int s = 0; s < KS; s++) {
                    half8 ka[2];
#pragma unroll
                    for (int tt = 0; tt < 2; tt++) ka[tt] = __builtin_bit_cast(half8, kp[(tt * KS + s) * 64]);
                    if constexpr (LOW) qf[NQ - 1][s] = s_low[s * 64];
#pragma unroll
                    for (int p = 0; p < NQ; p++)
#pragma unroll
                        for (int tt = 0; tt < 2; tt++)
                            c[tt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
                                ka[tt], __builtin_bit_cast(half8, qf[p][s]), c[tt], 0, 0, 0);
                }
            }
            read_ahead<(LOW ? 3 : 2) * KS, LOW ? 1 : NQ>();
            // exponents' factors and offsets by unit; l's weights
            float f[4], off[4], weight[4];
            if constexpr (I8) {
                const float vmax = fmaxf(fmaxf(vs[0], vs[1]), fmaxf(vs[2], vs[3]));
                if (vmax > U) {
                    const float k = U / vmax;
#pragma unroll
                    for (int d = 0; d < NS; d++) acc[d] *= k;
                    U = vmax;
                    log_U = __builtin_amdgcn_logf(U);
                }
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    // codes of a page without values are zeros, in any scale;
                    // under 2^-60 of U none of them is left in f16
                    const float w = vs[u] > 0.0f
                                        ? fmaxf(__builtin_amdgcn_logf(vs[u]) - log_U, -60.0f)
                                        : 0.0f;
                    f[u] = mul * ks[u];
                    off[u] = 6.0f + w;
                    weight[u] = __builtin_amdgcn_exp2f(-w);
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
                for (int u = 0; u < 4; u++) {
                    const int see = have >> (16 * u) & 1 ? pos - (step * 64 + 16 * u + 4 * g) : -1;
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        if (8 * (e / 4) + e % 4 > see) c[u / 2][8 * (u & 1) + e] = -INFINITY;
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
#pragma unroll
            for (int u = 0; u < 4; u++) {
                half8 va[NS];
#pragma unroll
                for (int d = 0; d < NS; d++) va[d] = vp[(u * NS + d) * 64];
#pragma unroll
                for (int p = 0; p < NP; p++)
#pragma unroll
                    for (int d = 0; d < NS; d++)
                        acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va[d], pf[p][u], acc[d], 0, 0, 0);
            }
            read_ahead<4 * NS, NP>();
            if constexpr (!I8) {
                if (s_odd[wt][n % SLOTS]) {
                    // the rows that see a token whose value is not finite
                    const int last = min(pos - step * 64, 63);
                    const unsigned long long see = last < 0 ? 0 : ~0ull >> (63 - last);
#pragma unroll
                    for (int d = 0; d < NS; d++)
#pragma unroll
                        for (int e = 0; e < 16; e++)
                            if (s_bad[wt * SLOTS + n % SLOTS][32 * d + 8 * (e / 4) + 4 * g + e % 4] & see)
                                acc[d][e] = NAN;
                }
            }
        }
        if constexpr (TWICE) {
            if (n + 1 < turns) store(step + 1, n + 1, buf ^ 1);
            __syncthreads();
            send(step + 2);
        } else {
            __syncthreads();
        }
    }
    float unit = I8 ? U : 1.0f;  // of the sums
    if constexpr (WT > 1) {
        // the shares' sums, in units of 2^(their largest m); the buffers are
        // free since the last barrier
        constexpr int LD = 32 * NS + 4;
        float *const s_ml = reinterpret_cast<float *>(s_kv);  // [WT][M][2]
        float *const s_o = s_ml + WT * M * 2;                 // [WT / 2][M][LD]
        static_assert((WT * M * 2 + WT / 2 * M * LD) * 4 <= sizeof(s_kv), "the buffers hold the sums");
        const int mine = 32 * wr + row;
        l = pair_sum(l);
        if (g == 0) {
            s_ml[(wt * M + mine) * 2] = m;
            s_ml[(wt * M + mine) * 2 + 1] = l;
        }
        __syncthreads();
        float top = kNone;
#pragma unroll
        for (int w = 0; w < WT; w++) top = fmaxf(top, s_ml[(w * M + mine) * 2]);
        const float f = __builtin_amdgcn_exp2f(m - top) * unit;
        l = 0.0f;
#pragma unroll
        for (int w = 0; w < WT; w++)
            l = __builtin_fmaf(s_ml[(w * M + mine) * 2 + 1],
                               __builtin_amdgcn_exp2f(s_ml[(w * M + mine) * 2] - top), l);
        l *= 0.5f;  // pair_sum adds it up again
        m = top;
        unit = 1.0f;
#pragma unroll
        for (int d = 0; d < NS; d++) acc[d] *= f;
#pragma unroll
        for (int from = WT / 2; from >= 1; from /= 2) {
            if (wt >= from && wt < 2 * from) {
                float *o = s_o + ((wt - from) * M + mine) * LD + 4 * g;
#pragma unroll
                for (int d = 0; d < NS; d++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        *reinterpret_cast<floatx4 *>(o + 32 * d + 8 * e) =
                            floatx4{acc[d][4 * e], acc[d][4 * e + 1], acc[d][4 * e + 2], acc[d][4 * e + 3]};
            }
            __syncthreads();
            if (wt < from) {
                const float *o = s_o + (wt * M + mine) * LD + 4 * g;
#pragma unroll
                for (int d = 0; d < NS; d++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const floatx4 v = *reinterpret_cast<const floatx4 *>(o + 32 * d + 8 * e);
#pragma unroll
                        for (int k = 0; k < 4; k++) acc[d][4 * e + k] += v[k];
                    }
            }
            __syncthreads();
        }
        if (wt) return;
    }
    if (!valid) return;
    l = pair_sum(l);
    const int64_t orow = x.s.row0 + i;
    const int head = h * G + r % G;
    const bool part = WT > 1 && x.parts > 1;  // blocks of many rows share none
    const float inv = part ? unit : l == 0.0f ? 0.0f : unit / l;
    const int64_t at = (orow * a.H + head) * t.splits + split;
    const auto out = [&](auto put) {
#pragma unroll
        for (int d = 0; d < NS; d++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                put(32 * d + 8 * e + 4 * g, floatx4{acc[d][4 * e], acc[d][4 * e + 1], acc[d][4 * e + 2],
                                                    acc[d][4 * e + 3]} * inv);
    };
    const int64_t to = orow * t.ldo + (int64_t)head * a.hd;
    if (part)
        out([&](int dim, floatx4 o) { *reinterpret_cast<floatx4 *>(t.part_o + at * (32 * NS) + dim) = o; });
    else
        out([&](int dim, floatx4 o) { if (dim < a.hd) store4_any(ACT, t.out, to + dim, o); });
    if (part && g == 0) {
        t.part_ml[2 * at] = m;
        t.part_ml[2 * at + 1] = l;
    }
}

template <int ACT>
hipError_t prompt_launch(const KvArgs &a, const AttendArgs &t, int tiles, bool many, hipStream_t st) {
    const dim3 grid((unsigned)tiles * a.KVH, t.splits);
    const auto go = [&](auto kern, int waves) { hipLaunchKernelGGL(kern, grid, dim3(64 * waves), 0, st, a, t); };
    by_dims(a, [&](auto ns) {
        constexpr int NS = decltype(ns)::value, MANY = kManyRows<NS>, SHARES = kShares<NS>;
        if (many) a.i8 ? go(k_attend_prompt<ACT, true, NS, MANY, 1>, MANY) : go(k_attend_prompt<ACT, false, NS, MANY, 1>, MANY);
        else a.i8 ? go(k_attend_prompt<ACT, true, NS, 2, SHARES>, 2 * SHARES) : go(k_attend_prompt<ACT, false, NS, 2, SHARES>, 2 * SHARES);
    });
    if (many) return hipGetLastError();
    return a.hdp <= 128 ? attend_join<64, 64, kPromptLeast<kShares<4>>>(a, t, tiles, st)
                        : attend_join<64, 64, kPromptLeast<kShares<8>>>(a, t, tiles, st);
}

}  // namespace lcmoe
