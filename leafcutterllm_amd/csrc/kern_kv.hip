// Appending keys and values to a paged cache, and reading it back
// (lcmoe_kv_append_dev, lcmoe_kv_read_dev).  The layout is in kv_device.h.

#include "kv_device.h"

namespace lcmoe {
namespace {

__device__ __forceinline__ double wave_max(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmax(v, __shfl_xor(v, o, 64));
    return v;
}

// pages that a sequence's new tokens reach
__device__ __forceinline__ int pages_touched(const KvArgs &a, const Seq &s) {
    if (s.cnt <= 0) return 0;
    const int off = s.len0 & ((1 << a.plog) - 1);
    return ((off + s.cnt - 1) >> a.plog) + 1;
}

// The 8-bit code of y: to nearest, ties to even, infinities at the ends, NaN
// as 0 (the conversion saturates, and makes 0 of NaN; written as the
// instruction, since the language leaves both undefined).  The product is in 64
// bits, where the rounding of y * (1 / scale) cannot move a code that the exact
// quotient has.
__device__ __forceinline__ uint32_t code_of(double y, double inv) {
    int q;
    asm("v_cvt_i32_f64 %0, %1" : "=v"(q) : "v"(__builtin_rint(y * inv)));
    return (uint32_t)min(max(q, -127), 127);
}

// y rounded once: to f32 and, where that is not exact, to the neighbour whose
// last bit is odd, so that rounding to f16 sees on which side y is
__device__ __forceinline__ _Float16 f16_of(double y) {
    const float f = (float)y;
    const double r = y - (double)f;
    uint32_t u = __float_as_uint(f);
    if ((r > 0.0 || r < 0.0) && !(u & 1)) u += (r > 0.0) == (f > 0.0f) ? 1u : ~0u;
    return (_Float16)__uint_as_float(u);
}
// |y|, 0 where it is not finite
__device__ __forceinline__ double finite(double y) {
    return fabs(y) < INFINITY ? fabs(y) : 0.0;
}
__device__ __forceinline__ float finite(float y) {
    return fabsf(y) < INFINITY ? fabsf(y) : 0.0f;
}

// A key's dims c .. c + 7 and h + c .. h + c + 7 (h = head_dim / 2), rotated by
// (cos, sin) = cs[c .. c + 7], or as they are:
//   y[d] = x[d] cos - x[h + d] sin,  y[h + d] = x[d] sin + x[h + d] cos.
// Products of two f32 are exact in 64 bits.
template <int ACT>
__device__ __forceinline__ void rotated8(const void *src, int64_t e, int h, const float *cs,
                                         double (&lo)[8], double (&hi)[8]) {
    float x[8], z[8], t[16];
    load_n<ACT>(src, e, x);
    load_n<ACT>(src, e + h, z);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        t[2 * i] = 1.0f;
        t[2 * i + 1] = 0.0f;
    }
    if (cs) __builtin_memcpy(t, cs, 64);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const double c = t[2 * i], s = t[2 * i + 1], zs = z[i] * s, xs = x[i] * s;
        // without an angle what is not finite must not meet the zero
        lo[i] = x[i] * c - (cs ? zs : 0.0);
        hi[i] = (cs ? xs : 0.0) + z[i] * c;
    }
}

// An item of values is tokens 4 g .. + 3 of a unit in dims 32 p + 4 q .. + 3 and
// 32 p + 16 + 4 q .. + 3: for each of the 4 dims, so many values apart, 2 x 4
// tokens in a row of the unit's.
template <bool I8>
__device__ __forceinline__ int v_item(int hdp, int p, int g, int q, int &apart) {
    apart = I8 && 32 * p < (hdp & ~63) ? 16 : 8;
    return v_place<I8>(hdp, 4 * g, 32 * p + 4 * q);
}

// What bounds it: 4 prompts of 2001 tokens, 8 heads of 128, bf16 into 8 bits, 22
// us, 2.2 TB/s of what it must move: two passes and code to be fetched in one
// round of blocks; one token each of 16 sequences 6.9 us, a chain of dependent
// loads.  7001 tokens of 16 heads, f32 into f16, one pass, 43 us, 4.0 TB/s.
//
// One block: the new tokens of one page, one K/V head, keys (z = 0) or values
// (z = 1).  In 8 bits the page's scale S' = max(S, max |new| / 127), S = 0
// where the page's first token is new; codes that were there are moved to the
// new scale where it grew; the new ones follow.  One block owns a page's head,
// so nothing here depends on the order in which blocks run.  Lanes go over
// tokens first, so that what a wave writes is whole lines.
template <int ACT, bool I8>
__global__ __launch_bounds__(256) void k_kv_append(KvArgs a, const void *__restrict__ ksrc,
                                                   int64_t ldk, const void *__restrict__ vsrc,
                                                   int64_t ldv, const float *__restrict__ rope) {
    const int h = blockIdx.y, value = blockIdx.z, tid = threadIdx.x;
    int j = 0;
    const int b = find_tile(a, blockIdx.x, [&](const Seq &s) { return pages_touched(a, s); }, j);
    if (b < 0) return;
    const Seq s = sequence(a, b);
    const int P = 1 << a.plog, page_no = (s.len0 >> a.plog) + j;
    const int t0 = max(page_no << a.plog, s.len0) - s.len0;  // the page's new tokens [t0, t1)
    const int t1 = min(s.cnt, ((page_no + 1) << a.plog) - s.len0);
    const int n = t1 - t0, slot0 = (s.len0 + t0) & (P - 1);
    const int page = a.pages[(int64_t)b * a.max_pages + page_no];
    if (page < 0 || page >= a.n_pages) return;
    const int hd = a.hd, hdp = a.hdp, half = hd / 2, row0 = s.row0 + t0;
    const void *src = value ? vsrc : ksrc;
    const int64_t ld = value ? ldv : ldk;
    const int64_t base = unit_base(a, page, h, 0);
    _Float16 *p16 = reinterpret_cast<_Float16 *>(value ? a.v : a.k) + base;
    uint8_t *p8 = (value ? a.v : a.k) + base;
    const int KC = half / 8, NB = hdp >> 5;  // 8-dim chunks of a key's half, 32-dim blocks
    const int unit0 = slot0 >> 4, units = ((slot0 + n + 15) >> 4) - unit0;
    // i / KC and i / NB of up to 16 * 16: exact
    const int by_kc = 65536 / KC + 1, by_nb = 65536 / NB + 1;
    double most = 0.0, inv = 0.0;
    // in 8 bits two turns, the first for the scale: one code for both, as a
    // line of code that is run once costs as much as it takes to fetch it
#pragma unroll 1
    for (int turn = I8 ? 0 : 1; turn < 2; turn++) {
        if (!value) {
#pragma unroll 1
            for (int i = tid >> 4; i < units * KC; i += 16) {
                const int u = (i * by_kc) >> 16, c = 8 * (i - u * KC);
                const int slot = (unit0 + u) * 16 + (tid & 15), t = slot - slot0;
                if (t < 0 || t >= n) continue;
                const int rot = (a.rope_abs ? s.len0 : 0) + t0 + t;
                double lo[8], hi[8];
                rotated8<ACT>(src, (int64_t)(row0 + t) * ld + (int64_t)h * hd + c, half,
                              rope ? rope + ((int64_t)rot * half + c) * 2 : nullptr, lo, hi);
                const int64_t at = (int64_t)(slot >> 4) * 16 * hdp;
                if constexpr (I8) {
                    if (!turn) {
#pragma unroll
                        for (int e = 0; e < 8; e++) most = fmax(most, fmax(finite(lo[e]), finite(hi[e])));
                        continue;
                    }
                    uintx2 wl, wh;
#pragma unroll
                    for (int e = 0; e < 8; e += 4) {
                        uint32_t ql[4], qh[4];
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            ql[k] = code_of(lo[e + k], inv);
                            qh[k] = code_of(hi[e + k], inv);
                        }
                        wl[e / 4] = bytes4<0>(ql);
                        wh[e / 4] = bytes4<0>(qh);
                    }
                    *reinterpret_cast<uintx2 *>(p8 + at + k_place<true>(hdp, slot & 15, c)) = wl;
                    *reinterpret_cast<uintx2 *>(p8 + at + k_place<true>(hdp, slot & 15, half + c)) = wh;
                } else {
                    half8 wl, wh;
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        wl[e] = f16_of(lo[e]);
                        wh[e] = f16_of(hi[e]);
                    }
                    *reinterpret_cast<half8 *>(p16 + at + k_place<false>(hdp, slot & 15, c)) = wl;
                    *reinterpret_cast<half8 *>(p16 + at + k_place<false>(hdp, slot & 15, half + c)) = wh;
                }
            }
        } else {
            // 16 items for each unit and 32 dims, the padding's zeros among them
#pragma unroll 1
            for (int i = tid; i < units * NB * 16; i += 256) {
                const int u = ((i >> 4) * by_nb) >> 16, p = (i >> 4) - u * NB, g = (i >> 2) & 3, q = i & 3;
                const int r0 = 16 * (unit0 + u) + 4 * g - slot0;  // the first of the item's 4 tokens
                if (r0 + 4 <= 0 || r0 >= n) continue;
                // every load in bounds and of the page's new rows: what a token
                // that is not new or a dim past the last brings is not kept
                const int d = 32 * p + 4 * q, d16 = d + 16 < hd ? d + 16 : d;
                float x[4][2][4];  // token, 16 dims, dim
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int64_t at = (int64_t)(row0 + min(max(r0 + e, 0), n - 1)) * ld + (int64_t)h * hd;
                    load_n<ACT>(src, at + min(d, hd - 4), x[e][0]);
                    load_n<ACT>(src, at + min(d16, hd - 4), x[e][1]);
                }
                if (I8 && !turn) {
                    float m = 0.0f;
#pragma unroll
                    for (int f = 0; f < 32; f++) m = fmaxf(m, finite(x[f >> 3][f >> 2 & 1][f & 3]));
                    most = fmax(most, (double)m);
                    continue;
                }
                // of tokens that are not new what is there stays
                using Word = std::conditional_t<I8, uint32_t, uint64_t>;
                constexpr int BITS = 2 * sizeof(Word);
                Word keep = 0;
                if (r0 < 0) keep |= ((Word)1 << BITS * -r0) - 1;
                if (r0 + 4 > n) keep |= ~(((Word)1 << BITS * (n - r0)) - 1);
                int apart;
                const int64_t at = (int64_t)(unit0 + u) * 16 * hdp + v_item<I8>(hdp, p, g, q, apart);
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    Word w[2], old[2];
                    Word *o = reinterpret_cast<Word *>(I8 ? (void *)(a.v + base + at + k * apart)
                                                          : (void *)(p16 + at + k * apart));
#pragma unroll
                    for (int t = 0; t < 2; t++) {
                        if constexpr (I8) {
                            uint32_t c[4];
#pragma unroll
                            for (int e = 0; e < 4; e++) c[e] = code_of(x[e][t][k], inv);
                            w[t] = bytes4<0>(c);
                        } else {
                            half4 c;
#pragma unroll
                            for (int e = 0; e < 4; e++) c[e] = (_Float16)x[e][t][k];
                            w[t] = __builtin_bit_cast(uint64_t, c);
                        }
                        if (d + 16 * t >= hd) w[t] = 0;
                    }
                    if (keep) {
                        __builtin_memcpy(old, __builtin_assume_aligned(o, sizeof(old)), sizeof(old));
                        w[0] = (w[0] & ~keep) | (old[0] & keep);
                        w[1] = (w[1] & ~keep) | (old[1] & keep);
                    }
                    __builtin_memcpy(__builtin_assume_aligned(o, sizeof(w)), w, sizeof(w));
                }
            }
        }
        if constexpr (I8) {
            if (turn) break;
            __shared__ double s_most[4];
            float *sp = a.scale + ((int64_t)page * a.KVH + h) * 2 + value;
            const float old = slot0 ? *sp : 0.0f;
            most = wave_max(most);
            if ((tid & 63) == 0) s_most[tid >> 6] = most;
            __syncthreads();
            most = fmax(fmax(s_most[0], s_most[1]), fmax(s_most[2], s_most[3]));
            const float scale = fmaxf(old, (float)(most / 127.0));
            inv = scale > 0.0f ? 1.0 / (double)scale : 0.0;
            if (slot0 && scale > old) {
                // every code of the units that hold old ones; what lies behind
                // them is written next, or is not read
                const double ratio = (double)old / (double)scale;
                const int words = ((slot0 + 15) >> 4) * 2 * hdp;
                uintx2 *w = reinterpret_cast<uintx2 *>(p8);
#pragma unroll 1
                for (int i = tid; i < words; i += 256) {
                    const uintx2 c = w[i];
                    uintx2 o = {0, 0};
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const int q = (int)__builtin_rint((double)(int8_t)(c[e >> 2] >> 8 * (e & 3)) * ratio);
                        o[e >> 2] |= (uint32_t)(uint8_t)q << 8 * (e & 3);
                    }
                    w[i] = o;
                }
            }
            __syncthreads();  // *sp read by every thread, the moved codes written
            if (tid == 0) *sp = scale;
        }
    }
    // the dims that pad a key to hdp meet zeros of the query: zeros too
    const int pad = value ? 0 : hdp - hd;
#pragma unroll 1
    for (int i = tid; i < pad * n; i += 256) {
        const int slot = slot0 + i / pad;
        const int64_t at = (int64_t)(slot >> 4) * 16 * hdp + k_place<I8>(hdp, slot & 15, hd + i % pad);
        if constexpr (I8) p8[at] = 0;
        else p16[at] = (_Float16)0.0f;
    }
}

// units of 16 tokens that a sequence's rows reach
__device__ __forceinline__ int units_touched(const Seq &s) {
    return s.cnt > 0 ? (((s.len0 & 15) + s.cnt - 1) >> 4) + 1 : 0;
}

// One block: one unit of 16 tokens, its K/V heads' items in turn, or a share of
// them where there are few units.  8 bits to bf16, 8176 tokens of 8 heads of 128:
// 11.6 us, 4.3 TB/s.
template <int ACT, bool I8>
__global__ __launch_bounds__(256) void k_kv_read(KvArgs a, void *__restrict__ ko, int64_t ldk,
                                                 void *__restrict__ vo, int64_t ldv) {
    int j = 0;
    const int b = find_tile(a, blockIdx.x, [&](const Seq &s) { return units_touched(s); }, j);
    if (b < 0) return;
    const Seq s = sequence(a, b);
    const int p0 = ((s.len0 >> 4) + j) << 4;  // the unit's first position
    const int page = a.pages[(int64_t)b * a.max_pages + (p0 >> a.plog)];
    const bool held = page >= 0 && page < a.n_pages;
    const int unit = (p0 & ((1 << a.plog) - 1)) >> 4, first = p0 - s.len0;
    const int hd = a.hd, hdp = a.hdp, C = hd / 8, NB = hdp >> 5;
    // keys: a token's 8 dims; values: items of 4 tokens
    const int KI = 16 * C, items = KI + 16 * NB;
    const auto scale_of = [&](int h, int value) {
        if (!held) return 0.0f;
        return I8 ? a.scale[((int64_t)page * a.KVH + h) * 2 + value] : 1.0f;
    };
    for (int i = blockIdx.y * 256 + threadIdx.x; i < a.KVH * items; i += 256 * gridDim.y) {
        const int h = i / items, k = i - h * items;
        const int64_t u = unit_base(a, held ? page : 0, h, unit);
        if (k < KI) {
            const int r = k & 15, d = 8 * (k >> 4), t = first + r;
            if (t < 0 || t >= s.cnt) continue;
            const float sc = scale_of(h, 0);
            float x[8];
            if constexpr (I8) {
                const uintx2 w = *reinterpret_cast<const uintx2 *>(a.k + u + k_place<true>(hdp, r, d));
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = (float)(int8_t)(w[e >> 2] >> 8 * (e & 3)) * sc;
            } else {
                const half8 w = *reinterpret_cast<const half8 *>(
                    reinterpret_cast<const _Float16 *>(a.k) + u + k_place<false>(hdp, r, d));
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = held ? (float)w[e] : 0.0f;
            }
            store_n<ACT>(ko, (int64_t)(s.row0 + t) * ldk + (int64_t)h * hd + d, x);
        } else {
            const int g = ((k - KI) >> 2) & 3, q = k & 3, t0 = first + 4 * g;
            if (t0 + 4 <= 0 || t0 >= s.cnt) continue;
            const float sc = scale_of(h, 1);
            const int p = (k - KI) >> 4;
            int apart;
            const int64_t at = u + v_item<I8>(hdp, p, g, q, apart);
            float x[4][2][4];  // token, 16 dims, dim
#pragma unroll
            for (int f = 0; f < 4; f++) {
                if constexpr (I8) {
                    const uintx2 w = *reinterpret_cast<const uintx2 *>(a.v + at + f * apart);
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        x[e & 3][e >> 2][f] = (float)(int8_t)(w[e >> 2] >> 8 * (e & 3)) * sc;
                } else {
                    const half8 w = *reinterpret_cast<const half8 *>(
                        reinterpret_cast<const _Float16 *>(a.v) + at + f * apart);
#pragma unroll
                    for (int e = 0; e < 8; e++) x[e & 3][e >> 2][f] = held ? (float)w[e] : 0.0f;
                }
            }
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (t0 + e < 0 || t0 + e >= s.cnt) continue;
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    const int d = 32 * p + 16 * t + 4 * q;
                    if (d < hd) store_n<ACT>(vo, (int64_t)(s.row0 + t0 + e) * ldv + (int64_t)h * hd + d, x[e][t]);
                }
            }
        }
    }
}

template <class F>
hipError_t by_type(int act, bool i8, F f) {
    switch (act) {
    case LCMOE_TYPE_F32: return i8 ? f(std::integral_constant<int, LCMOE_TYPE_F32>(), std::true_type()) : f(std::integral_constant<int, LCMOE_TYPE_F32>(), std::false_type());
    case LCMOE_TYPE_F16: return i8 ? f(std::integral_constant<int, LCMOE_TYPE_F16>(), std::true_type()) : f(std::integral_constant<int, LCMOE_TYPE_F16>(), std::false_type());
    default: return i8 ? f(std::integral_constant<int, LCMOE_TYPE_BF16>(), std::true_type()) : f(std::integral_constant<int, LCMOE_TYPE_BF16>(), std::false_type());
    }
}

}  // namespace

// a sequence of c new tokens touches at most (c - 1) / n + 2 blocks of n tokens
static int64_t most_blocks(const KvArgs &a, int n) {
    const int64_t each = (int64_t)(a.max_new + n - 2) / n + 1;
    return std::min((int64_t)a.n_rows / n + 2 * (int64_t)a.n_seq, each * a.n_seq);
}

hipError_t launch_kv_append(const KvArgs &a, const void *k, int64_t ldk, const void *v, int64_t ldv,
                            const float *rope, hipStream_t st) {
    const dim3 grid((unsigned)most_blocks(a, 1 << a.plog), a.KVH, 2);
    return by_type(a.act, a.i8, [&](auto act, auto i8) {
        hipLaunchKernelGGL((k_kv_append<decltype(act)::value, decltype(i8)::value>), grid, dim3(256),
                           0, st, a, k, ldk, v, ldv, rope);
        return hipGetLastError();
    });
}

hipError_t launch_kv_read(const KvArgs &a, void *k, int64_t ldk, void *v, int64_t ldv, hipStream_t st) {
    // heads of a unit over so many blocks that about 1024 run
    const int64_t tiles = most_blocks(a, 16);
    const int items = a.KVH * (2 * a.hd + (a.hdp + 31) / 32 * 16);
    const int64_t y = std::min<int64_t>((items + 255) / 256, std::max<int64_t>(1, 1024 / std::max<int64_t>(tiles, 1)));
    const dim3 grid((unsigned)tiles, (unsigned)std::min<int64_t>(y, 65535));
    return by_type(a.act, a.i8, [&](auto act, auto i8) {
        hipLaunchKernelGGL((k_kv_read<decltype(act)::value, decltype(i8)::value>), grid, dim3(256),
                           0, st, a, k, ldk, v, ldv);
        return hipGetLastError();
    });
}

}  // namespace lcmoe
