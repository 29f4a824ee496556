// The attention kernel over a paged cache, for both kinds of pages; its
// instances are in kern_kv_attn_i8.hip and kern_kv_attn_f16.hip, its launches
// in kern_kv_attn.hip.
//
// A block takes 16 query rows of one K/V head -- (token, query head of
// the group) pairs, so that grouped heads share the keys they read -- and a
// range of the context.  Its four waves take steps of ST tokens in turn, each
// with all M rows, and join at the end; blocks that share rows leave partials
// for k_attend_join.  A step is
//   S^T = K Q^T   [16 tokens x 16 rows] per unit of 16 tokens,
//   p = 2^(S - m) with the running maximum m and sum l,
//   O^T += V^T P^T  [16 dims x 16 rows] per 16 dims,
// all on 16x16 matrix instructions.  The lane that holds row r and tokens 4 g
// .. 4 g + 3 of a unit in S^T holds the same ones as an operand of P^T, so
// probabilities stay in registers; a unit's layout (kv_device.h) makes every
// operand of K and V a 16-byte load at lane * 16.
//
// 8-bit pages: codes go into integer products as they are (16x16x64, twice the
// f16 rate, no conversion).  Queries and probabilities become NP signed 8-bit
// pieces of a fixed-point value, x = sum of piece_i 256^i: 15 bits (NP = 2) of
// the row's largest for f16 and bf16 activations, 23 bits (NP = 3) for f32.
// Integer sums are exact; the scales are applied in f32, the keys' to the
// score, the values' to p, relative to the largest of the step.
// f16 pages: NP f16 pieces, of q scaled by a power of two, and of p 2^10.
//
// Bound by the cache's bytes where there are many: 64 sequences of 4096 in 8
// bits, 32 heads on 8 of 128, 70.5 us, 4.8 TB/s; one of 100,000 41 us, 5.0 TB/s,
// and 6.5 for the join.  One token on 500 is 7.2 us of latency and 3.5 of join.
// Sixteen rows are what the products take at least: a group of 4 heads fills a
// quarter of them, for nothing, as the matrix units have the time.
#pragma once

#include "kv_device.h"

namespace lcmoe {

struct AttendArgs {
    const void *q;
    int64_t ldq;
    const float *rope;
    float scale;
    void *out;
    int64_t ldo;
    int splits;   // blocks that may share a row
    int per_seq;  // tiles per sequence, all alike; 0: as many as its rows fill
    int lo, hi;   // sequences with lo < rows <= hi only (rows: tokens * group)
    float *part_o, *part_ml;
};

// tokens of a step, and the fewest steps that a block is given
template <bool I8> constexpr int kStep = I8 ? 64 : 32;
constexpr int kWaves = 4;

typedef int32_t intx4 __attribute__((ext_vector_type(4)));

// A tile of M rows of one sequence and its share of the context.
struct Tile {
    Seq s;
    int b, r0;       // sequence, first (token, head) row of the tile
    int rows;        // the sequence's rows
    int n_tok;       // tokens that some row of the tile sees
    int all_see;     // tokens that every row sees
    int steps, per, parts;  // steps, steps per block, blocks with any
};
// ST: tokens of a step; LEAST: steps that a block is worth
template <int ST, int M, int LEAST>
__device__ __forceinline__ bool find_rows(const KvArgs &a, const AttendArgs &t, int tile, Tile &x) {
    const int G = a.H / a.KVH;
    int j = 0;
    if (t.per_seq) {
        x.b = tile / t.per_seq;
        j = tile % t.per_seq;
    } else {
        x.b = find_tile(a, tile, [&](const Seq &s) {
            const int rows = max(s.cnt, 0) * G;
            return rows > t.lo && rows <= t.hi ? (rows + M - 1) / M : 0;
        }, j);
        if (x.b < 0) return false;
    }
    x.s = sequence(a, x.b);
    x.rows = max(x.s.cnt, 0) * G;
    x.r0 = j * M;
    if (x.r0 >= x.rows || x.rows <= t.lo || x.rows > t.hi) return false;
    x.all_see = x.s.len0 + x.r0 / G + 1;
    x.n_tok = x.s.len0 + (min(x.r0 + M, x.rows) - 1) / G + 1;
    x.steps = (x.n_tok + ST - 1) / ST;
    const int parts = min(t.splits, (x.steps + LEAST - 1) / LEAST);
    x.per = (x.steps + parts - 1) / parts;
    x.parts = (x.steps + x.per - 1) / x.per;
    return true;
}

// over the four lanes that hold a row (lane, lane ^ 16, ^ 32, ^ 48)
__device__ __forceinline__ float row_max(float v) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float row_sum(float v) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ void load8_any(int act, const void *p, int64_t e, float (&o)[8]) {
    if (act == LCMOE_TYPE_F32) load_n<LCMOE_TYPE_F32>(p, e, o);
    else if (act == LCMOE_TYPE_F16) load_n<LCMOE_TYPE_F16>(p, e, o);
    else load_n<LCMOE_TYPE_BF16>(p, e, o);
}
__device__ __forceinline__ void store4_any(int act, void *p, int64_t e, floatx4 v) {
    const float o[4] = {v[0], v[1], v[2], v[3]};
    if (act == LCMOE_TYPE_F32) store_n<LCMOE_TYPE_F32>(p, e, o);
    else if (act == LCMOE_TYPE_F16) store_n<LCMOE_TYPE_F16>(p, e, o);
    else store_n<LCMOE_TYPE_BF16>(p, e, o);
}

constexpr float kLog2e = 1.44269504088896340736f;

// f16 pieces of 8 values of a row whose largest is `most`, which comes to
// [2^14, 2^15), so that the pieces are normal f16 values
__device__ __forceinline__ int exponent_of(float most) {
    return most > 0.0f && most < INFINITY ? __builtin_amdgcn_frexp_expf(most) : 0;
}
template <int NP>
__device__ __forceinline__ void half_pieces(const float (&y)[8], int ex, half8 (&o)[NP]) {
#pragma unroll
    for (int k = 0; k < 8; k++) {
        const float v = __builtin_amdgcn_ldexpf(y[k], 15 - ex);
        o[0][k] = (_Float16)v;
        if constexpr (NP == 2) o[1][k] = (_Float16)(v - (float)o[0][k]);
    }
}

// The operands of one kind of page, for a head of 32 NS dims.  wide: 16-byte
// operands of 64 (8 bits) or 32 (f16) dims; tail: the last 32 in 8 bits.
template <bool I8, int NP, int NS>
struct Ops;

template <int NP, int NS>
struct Ops<true, NP, NS> {
    static constexpr int NJ = NS / 2, TAIL = NS & 1, UN = 4;
    static constexpr float kQ = NP == 2 ? 127.0f * 256 : 127.0f * 65536;  // most of x
    struct Unit {
        uintx4 w[NJ ? NJ : 1];
        uintx2 tail;
    };
    struct Row {  // one row's dims of the lane's group
        intx4 w[NP][NJ ? NJ : 1];
        int64_t tail[NP];
    };
    // a tile of 16 rows in LDS: [piece][64 dims][lane] of 16 bytes, then [piece][lane] of 8
    static constexpr int kTile = NP * (NJ * 1024 + TAIL * 512);
    __device__ __forceinline__ static void put(uint8_t *q, int row, int c, const float (&y)[8], float most) {
        uint32_t o0[NP], o1[NP];
        pieces(&y[0], most, o0);
        pieces(&y[4], most, o1);
        const bool wide = c < 8 * NJ;
        const int lane = (wide ? (c & 7) >> 1 : c & 3) * 16 + row;
        const int at = wide ? (c >> 3) * 1024 + lane * 16 + (c & 1) * 8 : NP * NJ * 1024 + lane * 8;
#pragma unroll
        for (int p = 0; p < NP; p++)
            *reinterpret_cast<uintx2 *>(q + at + p * (wide ? NJ * 1024 : 512)) = uintx2{o0[p], o1[p]};
    }
    __device__ __forceinline__ static float factor(float most, float scale) {
        return most * scale * (kLog2e / kQ);
    }
    __device__ __forceinline__ static void take(Row &r, const uint8_t *q, int lane) {
#pragma unroll
        for (int p = 0; p < NP; p++) {
#pragma unroll
            for (int j = 0; j < NJ; j++)
                r.w[p][j] = *reinterpret_cast<const intx4 *>(q + (p * NJ + j) * 1024 + lane * 16);
            if constexpr (TAIL != 0)
                r.tail[p] = *reinterpret_cast<const int64_t *>(q + NP * NJ * 1024 + p * 512 + lane * 8);
        }
    }
    __device__ __forceinline__ static void load(Unit &u, const uint8_t *p, int lane) {
#pragma unroll
        for (int j = 0; j < NJ; j++)
            u.w[j] = *reinterpret_cast<const uintx4 *>(p + j * 1024 + lane * 16);
        if constexpr (TAIL != 0)
            u.tail = *reinterpret_cast<const uintx2 *>(p + NJ * 1024 + lane * 8);
    }
    // pieces of y / most, |y| <= most, for 4 values: piece NP - 1 the lowest
    __device__ __forceinline__ static void pieces(const float *y, float most, uint32_t (&o)[NP]) {
        uint32_t x[4], c[4];
        const int ex = exponent_of(most);
        const float to = most > 0.0f ? kQ / __builtin_amdgcn_ldexpf(most, -ex) : 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++)
            x[i] = (uint32_t)(int32_t)__builtin_rintf(__builtin_amdgcn_ldexpf(y[i], -ex) * to);
        o[NP - 1] = bytes4<0>(x);
#pragma unroll
        for (int i = 0; i < 4; i++) c[i] = x[i] + 128u;
        o[NP - 2] = bytes4<1>(c);
        if constexpr (NP == 3) {
#pragma unroll
            for (int i = 0; i < 4; i++) c[i] = x[i] + 128u + 32768u;
            o[0] = bytes4<2>(c);
        }
    }
};

template <int NP, int NS>
struct Ops<false, NP, NS> {
    static constexpr int NJ = NS, TAIL = 0, UN = 2;
    struct Unit {
        half8 w[NJ];
    };
    struct Row {
        half8 w[NP][NJ];
    };
    // a tile of 16 rows in LDS: [piece][32 dims][lane] of 16 bytes
    static constexpr int kTile = NP * NJ * 1024;
    __device__ __forceinline__ static void put(uint8_t *q, int row, int c, const float (&y)[8], float most) {
        half8 o[NP];
        half_pieces<NP>(y, exponent_of(most), o);
#pragma unroll
        for (int p = 0; p < NP; p++)
            *reinterpret_cast<half8 *>(q + (p * NJ + (c >> 2)) * 1024 + ((c & 3) * 16 + row) * 16) = o[p];
    }
    __device__ __forceinline__ static float factor(float most, float scale) {
        return __builtin_amdgcn_ldexpf(scale, exponent_of(most) - 15) * kLog2e;
    }
    __device__ __forceinline__ static void take(Row &r, const uint8_t *q, int lane) {
#pragma unroll
        for (int p = 0; p < NP; p++)
#pragma unroll
            for (int j = 0; j < NJ; j++)
                r.w[p][j] = *reinterpret_cast<const half8 *>(q + (p * NJ + j) * 1024 + lane * 16);
    }
    __device__ __forceinline__ static void load(Unit &u, const uint8_t *p, int lane) {
#pragma unroll
        for (int j = 0; j < NJ; j++)
            u.w[j] = *reinterpret_cast<const half8 *>(p + j * 1024 + lane * 16);
    }
};

// A tile's rows of q, rotated, once for a block of T threads: every thread
// takes 8 dims of a row at a time, as many neighbours as a row has (rounded up
// to a power of two) find its largest magnitude, and put(row, d / 8, y, most)
// keeps the 8 values; per row keep(row, most, bad), bad NaN where a value is not
// finite.  Rows past the sequence's last are zeros.  One loop, for its code is
// run once and fetched for it.
template <int NS, int M, int T, class Load, class Put, class Keep>
__device__ __forceinline__ void stage_q(const KvArgs &a, const AttendArgs &t, const Tile &x, int h,
                                        Load load, Put put, Keep keep) {
    constexpr int C = 4 * NS, L = C <= 4 ? 4 : C <= 8 ? 8 : C <= 16 ? 16 : 32;  // lanes of a row
    const int G = a.H / a.KVH, half = a.hd / 2, d = 8 * (threadIdx.x & (L - 1));
#pragma unroll 1
    for (int r = threadIdx.x / L; r < M; r += T / L) {
        const int rr = x.r0 + r, i = rr / G;
        float y[8], z[8], most = 0.0f, bad = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; k++) y[k] = 0.0f;
        if (rr < x.rows && d < a.hd) {
            const int64_t e = (int64_t)(x.s.row0 + i) * t.ldq + (int64_t)(h * G + rr - i * G) * a.hd;
            load(e + d, y);
            if (t.rope) {
                const bool up = d >= half;
                const int o = up ? d - half : d;
                load(e + (up ? o : d + half), z);
                const float *w = t.rope + (int64_t)(a.rope_abs ? x.s.len0 + i : i) * a.hd + 2 * o;
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const float c = w[2 * k], s = up ? -w[2 * k + 1] : w[2 * k + 1];
                    y[k] = y[k] * c - z[k] * s;
                }
            }
        }
#pragma unroll
        for (int k = 0; k < 8; k++) {
            most = fmaxf(most, fabsf(y[k]));
            bad = __builtin_fmaf(y[k], 0.0f, bad);
        }
#pragma unroll
        for (int o = 1; o < L; o <<= 1) {
            most = fmaxf(most, __shfl_xor(most, o, 64));
            bad += __shfl_xor(bad, o, 64);
        }
        if (d < 8 * C) put(r, d >> 3, y, most);
        if (d == 0) keep(r, most, bad);
    }
}

template <bool I8, int NP, int NS>
__global__ __launch_bounds__(256) void k_attend(KvArgs a, AttendArgs t) {
    typedef Ops<I8, NP, NS> O;
    constexpr int M = 16, HDP = 32 * NS, UN = O::UN, ST = kStep<I8>, TD = HDP / 16;
    constexpr int LD = HDP + 4, kSums = kWaves * M * LD * 4;
    // the rows of q, then the four waves' sums
    __shared__ __attribute__((aligned(16))) uint8_t s_mem[kSums > O::kTile ? kSums : O::kTile];
    __shared__ float s_mul[M], s_m[kWaves][M], s_l[kWaves][M];
    const int lane = threadIdx.x & 63, grp = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = blockIdx.x % a.KVH, split = blockIdx.y, G = a.H / a.KVH;
    Tile x;
    // the last tiles first: a prompt's see the most
    if (!find_rows<ST, M, kWaves>(a, t, gridDim.x / a.KVH - 1 - blockIdx.x / a.KVH, x)) return;
    if (split >= x.parts) return;
    const int step0 = split * x.per + wave, step1 = min(x.steps, (split + 1) * x.per);
    const int last_unit = (x.n_tok - 1) >> 4, ushift = a.plog - 4;
    const int32_t *table = a.pages + (int64_t)x.b * a.max_pages;
    // of the next 64 units that this wave meets, one a lane: whether their page
    // is there, its scales, and the unit's place in the pools
    int m_there = 0;
    float m_ks = 0.0f, m_vs = 0.0f;
    uint32_t m_lo = 0, m_hi = 0;
    const auto fetch_meta = [&](int step) {
        const int unit = min((step + kWaves * (lane / UN)) * UN + lane % UN, last_unit);
        int page = table[unit >> ushift];
        m_there = page >= 0 && page < a.n_pages;
        page = m_there ? page : 0;
        const int64_t at = unit_base(a, page, h, unit & ((1 << ushift) - 1)) * (I8 ? 1 : 2);
        m_lo = (uint32_t)at;
        m_hi = (uint32_t)(at >> 32);
        if constexpr (I8) {
            const float *s = a.scale + ((int64_t)page * a.KVH + h) * 2;
            m_ks = m_there ? s[0] : 0.0f;
            m_vs = m_there ? s[1] : 0.0f;
        }
    };
    // unit u of the step `in` steps after the fetch
    const auto load = [&](typename O::Unit &w, const uint8_t *pool, int in, int u) {
        const uint64_t at = (uint32_t)__builtin_amdgcn_readlane(m_lo, in * UN + u) |
                            (uint64_t)(uint32_t)__builtin_amdgcn_readlane(m_hi, in * UN + u) << 32;
        O::load(w, pool + at, lane);
    };
    typename O::Unit kf[UN], vf[UN];
    int in = 0;
    fetch_meta(step0);
#pragma unroll
    for (int u = 0; u < UN; u++) load(kf[u], a.k, 0, u);

    stage_q<NS, M, 256>(a, t, x, h,
        [&](int64_t e, float (&y)[8]) { load8_any(a.act, t.q, e, y); },
        [&](int row, int c, const float (&y)[8], float most) { O::put(s_mem, row, c, y, most); },
        [&](int row, float most, float bad) { s_mul[row] = O::factor(most, t.scale) + bad; });
    __syncthreads();
    typename O::Row qf;
    O::take(qf, s_mem, lane);
    const float mul = s_mul[lane & 15];
    // rows past the last see every token and are not stored
    const int r_own = x.r0 + (lane & 15), pos = r_own < x.rows ? x.s.len0 + r_own / G : 0x7fffffff;
    __syncthreads();  // s_mem is the sums' from here on

    floatx4 acc[TD];
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int d = 0; d < TD; d++) acc[d] = floatx4{0, 0, 0, 0};
    for (int step = step0; step < step1; step += kWaves) {
        bool there[UN];
        float ks[UN], vs[UN];
        bool whole = (step + 1) * ST <= x.all_see;
#pragma unroll
        for (int u = 0; u < UN; u++) {
            there[u] = __builtin_amdgcn_readlane(m_there, in * UN + u) != 0;
            whole = whole && there[u];
            if constexpr (I8) {
                ks[u] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(m_ks), in * UN + u));
                vs[u] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(m_vs), in * UN + u));
            }
            load(vf[u], a.v, in, u);
        }
        // scores
        float s[UN][4];
#pragma unroll
        for (int u = 0; u < UN; u++) {
            if constexpr (I8) {
                intx4 c[NP];
#pragma unroll
                for (int p = 0; p < NP; p++) {
                    c[p] = intx4{0, 0, 0, 0};
#pragma unroll
                    for (int j = 0; j < O::NJ; j++)
                        c[p] = __builtin_amdgcn_mfma_i32_16x16x64_i8(
                            __builtin_bit_cast(intx4, kf[u].w[j]), qf.w[p][j], c[p], 0, 0, 0);
                    if constexpr (O::TAIL != 0)
                        c[p] = __builtin_amdgcn_mfma_i32_16x16x32_i8(
                            __builtin_bit_cast(int64_t, kf[u].tail), qf.tail[p], c[p], 0, 0, 0);
                }
                const float f = mul * ks[u];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    // |low two| < 2^31: 256 dims of 127 * 127 times 257
                    float v = (float)((c[NP - 2][e] << 8) + c[NP - 1][e]);
                    if constexpr (NP == 3) v = __builtin_fmaf((float)c[0][e], 65536.0f, v);
                    s[u][e] = v * f;
                }
            } else {
                floatx4 c = {0, 0, 0, 0};
#pragma unroll
                for (int p = 0; p < NP; p++)
#pragma unroll
                    for (int j = 0; j < O::NJ; j++)
                        c = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[u].w[j], qf.w[p][j], c, 0, 0, 0);
#pragma unroll
                for (int e = 0; e < 4; e++) s[u][e] = c[e] * mul;
            }
        }
        // the next step's keys go out before this one's softmax
        if (step + kWaves < step1) {
            in++;
            if (in == 64 / UN) {
                in = 0;
                fetch_meta(step + kWaves);
            }
#pragma unroll
            for (int u = 0; u < UN; u++) load(kf[u], a.k, in, u);
        }
        bool odd = false;
        if (!whole) {
#pragma unroll
            for (int u = 0; u < UN; u++) {
                const int tok = step * ST + 16 * u + 4 * grp;
                const int see = there[u] ? min(pos, x.n_tok - 1) - tok : -1;
#pragma unroll
                for (int e = 0; e < 4; e++) s[u][e] = e <= see ? s[u][e] : -INFINITY;
                if constexpr (!I8) {
                    // what no row sees may be NaN, and would meet a p of zero
                    const int n = there[u] ? min(max(x.n_tok - tok, 0), 4) : 0;
                    const uint64_t keep = n == 4 ? ~0ull : (1ull << 16 * n) - 1;
                    half8 z = {};
#pragma unroll
                    for (int j = 0; j < O::NJ; j++) {
                        uintx4 w = __builtin_bit_cast(uintx4, vf[u].w[j]);
                        w &= uintx4{(uint32_t)keep, (uint32_t)(keep >> 32), (uint32_t)keep, (uint32_t)(keep >> 32)};
                        vf[u].w[j] = __builtin_bit_cast(half8, w);
                        z += vf[u].w[j] * (_Float16)0.0f;
                    }
#pragma unroll
                    for (int k = 0; k < 8; k++) odd = odd || z[k] != z[k];
                }
            }
            if constexpr (!I8) odd = __ballot(odd) != 0;
        }
        float vmax = 0.0f, vmul = 0.0f, ratio[UN];
        if constexpr (I8) {
#pragma unroll
            for (int u = 0; u < UN; u++) vmax = fmaxf(vmax, vs[u]);
            // a reciprocal that neither overflows nor is lost
            const float big = vmax < 0x1p-100f ? 0x1p100f : 1.0f;
            const float inv = vmax > 0.0f ? __builtin_amdgcn_rcpf(vmax * big) : 0.0f;
#pragma unroll
            for (int u = 0; u < UN; u++) ratio[u] = vs[u] * big * inv * O::kQ;
            vmul = vmax * (1.0f / O::kQ);
        }
        float mx = -INFINITY;
#pragma unroll
        for (int u = 0; u < UN; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) mx = fmaxf(mx, s[u][e]);
        mx = fmaxf(m, row_max(mx));
        const float base = mx == -INFINITY ? 0.0f : mx;
        const float keep = __builtin_amdgcn_exp2f(m - base);
        m = mx;
        float sum = 0.0f;
#pragma unroll
        for (int u = 0; u < UN; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                s[u][e] = __builtin_amdgcn_exp2f(s[u][e] - (I8 ? base : base - 10.0f));
                sum += s[u][e];
            }
        l = __builtin_fmaf(l, keep, sum);
        if (__ballot(keep != 1.0f)) {
#pragma unroll
            for (int d = 0; d < TD; d++) acc[d] *= keep;
        }
        if constexpr (I8) {
            intx4 pf[NP];
#pragma unroll
            for (int u = 0; u < UN; u++) {
                uint32_t b[4], c[4];
#pragma unroll
                for (int e = 0; e < 4; e++)  // the fraction's bits: p ratio, rounded
                    b[e] = __float_as_uint(__builtin_fmaf(s[u][e], ratio[u], 8388608.0f));
                pf[NP - 1][u] = (int)bytes4<0>(b);
#pragma unroll
                for (int e = 0; e < 4; e++) c[e] = b[e] + 128u;
                pf[NP - 2][u] = (int)bytes4<1>(c);
                if constexpr (NP == 3) {
#pragma unroll
                    for (int e = 0; e < 4; e++) c[e] = b[e] + 128u + 32768u;
                    pf[0][u] = (int)bytes4<2>(c);
                }
            }
#pragma unroll
            for (int d = 0; d < TD; d++) {
                intx4 va, c[NP];
#pragma unroll
                for (int u = 0; u < UN; u++)
                    va[u] = d < 4 * O::NJ ? (int)vf[u].w[O::NJ ? d / 4 : 0][d % 4]
                                          : (int)vf[u].tail[d % 2];
#pragma unroll
                for (int p = 0; p < NP; p++)
                    c[p] = __builtin_amdgcn_mfma_i32_16x16x64_i8(va, pf[p], intx4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float v = (float)((c[NP - 2][e] << 8) + c[NP - 1][e]);
                    acc[d][e] = __builtin_fmaf(v, vmul, acc[d][e]);
                    if constexpr (NP == 3)
                        acc[d][e] = __builtin_fmaf((float)c[0][e], vmul * 65536.0f, acc[d][e]);
                }
            }
        } else {
            half8 pf[NP];
#pragma unroll
            for (int u = 0; u < UN; u++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const _Float16 hi = (_Float16)s[u][e];
                    pf[0][4 * u + e] = hi;
                    if constexpr (NP == 2) pf[1][4 * u + e] = (_Float16)(s[u][e] - (float)hi);
                }
            if (odd) {
                // values that are not finite meet only the rows that see them,
                // whose sums they leave NaN
                half8 see;
#pragma unroll
                for (int k = 0; k < 8; k++)
                    see[k] = step * ST + 16 * (k / 4) + 4 * grp + k % 4 <= pos ? (_Float16)1.0f
                                                                             : (_Float16)0.0f;
#pragma unroll
                for (int d = 0; d < TD; d++) {
                    half8 is;
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        const _Float16 v = vf[k / 4].w[d / 2][4 * (d % 2) + k % 4];
                        const _Float16 z = v * (_Float16)0.0f;
                        is[k] = z == z ? (_Float16)0.0f : (_Float16)1.0f;
                        if (z != z) vf[k / 4].w[d / 2][4 * (d % 2) + k % 4] = (_Float16)0.0f;
                    }
                    const floatx4 c = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                        is, see, floatx4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (c[e] > 0.0f) acc[d][e] = NAN;
                }
            }
#pragma unroll
            for (int d = 0; d < TD; d++) {
                half8 va;
#pragma unroll
                for (int u = 0; u < UN; u++)
#pragma unroll
                    for (int e = 0; e < 4; e++) va[4 * u + e] = vf[u].w[d / 2][4 * (d % 2) + e];
#pragma unroll
                for (int p = 0; p < NP; p++)
                    acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pf[p], acc[d], 0, 0, 0);
            }
        }
    }

    // the four waves' sums, in units of 2^(their largest maximum)
    float *const s_o = reinterpret_cast<float *>(s_mem);
    l = row_sum(l);
    if (lane < 16) {
        s_m[wave][lane] = m;
        s_l[wave][lane] = l;
    }
#pragma unroll
    for (int d = 0; d < TD; d++)
        *reinterpret_cast<floatx4 *>(s_o + (wave * M + (lane & 15)) * LD + 16 * d + 4 * grp) = acc[d];
    __syncthreads();
    const int C = (x.parts == 1 ? a.hd : HDP) / 4;
#pragma unroll 1
    for (int k = threadIdx.x; k < M * C; k += 256) {
        const int i = k / C, d = 4 * (k - i * C), r = x.r0 + i;
        if (r >= x.rows) break;
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; w++) top = fmaxf(top, s_m[w][i]);
        const float base = top == -INFINITY ? 0.0f : top;
        floatx4 o = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            const float f = __builtin_amdgcn_exp2f(s_m[w][i] - base);
            sum = __builtin_fmaf(s_l[w][i], f, sum);
            o += *reinterpret_cast<const floatx4 *>(s_o + (w * M + i) * LD + d) * f;
        }
        const int64_t row = x.s.row0 + r / G;
        const int head = h * G + r % G;
        if (x.parts == 1) {
            store4_any(a.act, t.out, row * t.ldo + (int64_t)head * a.hd + d,
                       o * (sum == 0.0f ? 0.0f : 1.0f / sum));
        } else {
            const int64_t at = (row * a.H + head) * t.splits + split;
            *reinterpret_cast<floatx4 *>(t.part_o + at * HDP + d) = o;
            if (d == 0) {
                t.part_ml[2 * at] = top;
                t.part_ml[2 * at + 1] = sum;
            }
        }
    }
}

// Rows that several blocks shared: their sums in units of 2^(the largest
// maximum).  A block takes one row; groups of hdp / 4 threads, four dims each,
// take the parts in turn and add up in LDS.
template <int ST, int M, int LEAST>
__global__ __launch_bounds__(256) void k_attend_join(KvArgs a, AttendArgs t) {
    __shared__ __attribute__((aligned(16))) floatx4 s_o[256];
    __shared__ float s_f[128];
    const int h = blockIdx.x % a.KVH, G = a.H / a.KVH, tid = threadIdx.x;
    Tile x;
    if (!find_rows<ST, M, LEAST>(a, t, gridDim.x / a.KVH - 1 - blockIdx.x / a.KVH, x)) return;
    const int r = x.r0 + blockIdx.y;
    if (x.parts == 1 || r >= x.rows) return;
    const int64_t row = x.s.row0 + r / G;
    const int head = h * G + r % G;
    const int64_t at = (row * a.H + head) * t.splits;
    // every wave for itself, two of at most 128 parts a lane: their largest
    // maximum, their factors, and the sum of their sums
    float mp[2], lp[2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const int s = (tid & 63) + 64 * k;
        mp[k] = s < x.parts ? t.part_ml[2 * (at + s)] : -INFINITY;
        lp[k] = s < x.parts ? t.part_ml[2 * (at + s) + 1] : 0.0f;
    }
    float top = fmaxf(mp[0], mp[1]);
    const int lanes = min(x.parts, 64);  // that hold any; the first has their sums
#pragma unroll 1
    for (int o = 1; o < lanes; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    const float base = top == -INFINITY ? 0.0f : top;
    float l = 0.0f;
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const float f = __builtin_amdgcn_exp2f(mp[k] - base);
        if (tid < 64) s_f[tid + 64 * k] = f;
        l = __builtin_fmaf(lp[k], f, l);
    }
#pragma unroll 1
    for (int o = 1; o < lanes; o <<= 1) l += __shfl_xor(l, o, 64);
    l = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(l)));
    __syncthreads();
    const int C = a.hdp / 4, groups = 256 / C, grp = tid / C, d = 4 * (tid % C);
    floatx4 o = {0, 0, 0, 0};
    if (grp < groups) {
        const float *p = t.part_o + at * a.hdp + d;
#pragma unroll 4
        for (int s = grp; s < x.parts; s += groups)
            o += *reinterpret_cast<const floatx4 *>(p + (int64_t)s * a.hdp) * s_f[s];
    }
    s_o[tid] = o;
    __syncthreads();
    if (grp || d >= a.hd) return;
    for (int k = 1; k < groups; k++) o += s_o[k * C + tid];
    store4_any(a.act, t.out, row * t.ldo + (int64_t)head * a.hd + d,
               o * (l == 0.0f ? 0.0f : 1.0f / l));
}

// Launches over `tiles` tiles: of 16 rows (attend_*), or of many (kManyRows * 32)
// or 64 rows (prompt_*), with the join where blocks share rows.
hipError_t attend_i8(const KvArgs &a, const AttendArgs &t, int tiles, hipStream_t st);
hipError_t attend_f16(const KvArgs &a, const AttendArgs &t, int tiles, hipStream_t st);
hipError_t prompt_f32(const KvArgs &a, const AttendArgs &t, int tiles, bool many, hipStream_t st);
hipError_t prompt_f16(const KvArgs &a, const AttendArgs &t, int tiles, bool many, hipStream_t st);
hipError_t prompt_bf16(const KvArgs &a, const AttendArgs &t, int tiles, bool many, hipStream_t st);

template <int ST, int M, int LEAST>
hipError_t attend_join(const KvArgs &a, const AttendArgs &t, int tiles, hipStream_t st) {
    if (t.splits > 1)
        hipLaunchKernelGGL((k_attend_join<ST, M, LEAST>), dim3((unsigned)tiles * a.KVH, M), dim3(256),
                           0, st, a, t);
    return hipGetLastError();
}

// f(the head's 32 dims, as a constant)
template <class F>
void by_dims(const KvArgs &a, F f) {
    switch (a.hdp / 32) {
    case 1: f(std::integral_constant<int, 1>()); break;
    case 2: f(std::integral_constant<int, 2>()); break;
    case 3: f(std::integral_constant<int, 3>()); break;
    case 4: f(std::integral_constant<int, 4>()); break;
    case 6: f(std::integral_constant<int, 6>()); break;
    default: f(std::integral_constant<int, 8>()); break;
    }
}

template <bool I8, int NP>
hipError_t attend_launch(const KvArgs &a, const AttendArgs &t, int tiles, hipStream_t st) {
    by_dims(a, [&](auto ns) {
        hipLaunchKernelGGL((k_attend<I8, NP, decltype(ns)::value>),
                           dim3((unsigned)tiles * a.KVH, t.splits), dim3(256), 0, st, a, t);
    });
    return attend_join<kStep<I8>, 16, kWaves>(a, t, tiles, st);
}

}  // namespace lcmoe
