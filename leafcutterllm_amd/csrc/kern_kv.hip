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
// as 0.  The product is in 64 bits, where the rounding of y * (1 / scale)
// cannot move a code that the exact quotient has.
__device__ __forceinline__ int code_of(double y, double inv) {
    const double q = __builtin_rint(y * inv);
    return q == q ? (int)fmin(fmax(q, -127.0), 127.0) : 0;
}

// f(i, y[c + i], y[h + c + i]) for a key's dims c .. c + 7 and h + c .. h + c +
// 7 (h = head_dim / 2), rotated by (cos, sin) = rope[c .. c + 7]:
//   y[d] = x[d] cos - x[h + d] sin,  y[h + d] = x[d] sin + x[h + d] cos.
// Products of two f32 are exact in 64 bits.
template <int ACT, class F>
__device__ __forceinline__ void rotated8(const void *src, int64_t e, int h, const float *cs, F f) {
    float x[8], z[8];
    load_n<ACT>(src, e, x);
    load_n<ACT>(src, e + h, z);
    float t[16];
    if (cs) __builtin_memcpy(t, cs, 64);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const double c = t[2 * i], s = t[2 * i + 1];
        if (cs) f(i, x[i] * c - z[i] * s, x[i] * s + z[i] * c);
        else f(i, (double)x[i], (double)z[i]);
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

// What bounds it: 4 prompts of 2001 tokens, 8 heads of 128, bf16 into 8 bits, 24
// us, 1.4 TB/s of what it must move: two passes, and 64-bit arithmetic; one
// token each of 16 sequences 7.6 us, a chain of dependent loads.  7001 tokens of
// 16 heads, f32 into f16, one pass, 61 us, 2.9 TB/s.
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
    const int KC = half / 8;  // 8-dim chunks of a key's half
    const int unit0 = slot0 >> 4, units = ((slot0 + n + 15) >> 4) - unit0;
    // item i of the units' keys: a slot and its chunk, if it is one of the new
    const auto key_at = [&](int i, int &slot, int &c) {
        const int u = i / (16 * KC);
        c = 8 * ((i - u * 16 * KC) >> 4);
        slot = (unit0 + u) * 16 + (i & 15);
        return slot >= slot0 && slot < slot0 + n;
    };
    const auto key8 = [&](int slot, int c, auto f) {
        const int t = slot - slot0, rot = (a.rope_abs ? s.len0 : 0) + t0 + t;
        rotated8<ACT>(src, (int64_t)(row0 + t) * ld + (int64_t)h * hd + c, half,
                      rope ? rope + ((int64_t)rot * half + c) * 2 : nullptr, f);
    };
    double inv = 0.0;
    if constexpr (I8) {
        float *sp = a.scale + ((int64_t)page * a.KVH + h) * 2 + value;
        const float old = slot0 ? *sp : 0.0f;
        double most = 0.0;
        const auto larger = [&](double y) {
            const double m = fabs(y);
            if (m > most && m < INFINITY) most = m;
        };
        if (!value) {
            for (int i = tid; i < units * 16 * KC; i += 256) {
                int slot, c;
                if (key_at(i, slot, c))
                    key8(slot, c, [&](int, double lo, double hi) {
                        larger(lo);
                        larger(hi);
                    });
            }
        } else {
            const int C = hd / 8;
            for (int i = tid; i < n * C; i += 256) {
                float x[8];
                load_n<ACT>(src, (int64_t)(row0 + i / C) * ld + (int64_t)h * hd + 8 * (i % C), x);
#pragma unroll
                for (int e = 0; e < 8; e++) larger(x[e]);
            }
        }
        __shared__ double s_most[4];
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
    if (!value) {
        for (int i = tid; i < units * 16 * KC; i += 256) {
            int slot, c;
            if (!key_at(i, slot, c)) continue;
            const int64_t u = (int64_t)(slot >> 4) * 16 * hdp;
            if constexpr (I8) {
                uintx2 wl = {0, 0}, wh = {0, 0};
                key8(slot, c, [&](int e, double lo, double hi) {
                    wl[e >> 2] |= (uint32_t)(uint8_t)code_of(lo, inv) << 8 * (e & 3);
                    wh[e >> 2] |= (uint32_t)(uint8_t)code_of(hi, inv) << 8 * (e & 3);
                });
                *reinterpret_cast<uintx2 *>(p8 + u + k_place<true>(hdp, slot & 15, c)) = wl;
                *reinterpret_cast<uintx2 *>(p8 + u + k_place<true>(hdp, slot & 15, half + c)) = wh;
            } else {
                half8 wl, wh;
                key8(slot, c, [&](int e, double lo, double hi) {
                    wl[e] = (_Float16)lo;
                    wh[e] = (_Float16)hi;
                });
                *reinterpret_cast<half8 *>(p16 + u + k_place<false>(hdp, slot & 15, c)) = wl;
                *reinterpret_cast<half8 *>(p16 + u + k_place<false>(hdp, slot & 15, half + c)) = wh;
            }
        }
        // the dims that pad the head to hdp meet zeros of the query: zeros too
        if (const int pad = hdp - hd)
            for (int i = tid; i < pad * n; i += 256) {
                const int slot = slot0 + i / pad;
                const int64_t at = (int64_t)(slot >> 4) * 16 * hdp +
                                   k_place<I8>(hdp, slot & 15, hd + i % pad);
                if constexpr (I8) p8[at] = 0;
                else p16[at] = (_Float16)0.0f;
            }
        return;
    }
    // values: 16 items for each unit and 32 dims, the padding's zeros among them
    const int NB = hdp >> 5;
    for (int i = tid; i < units * NB * 16; i += 256) {
        const int u = i / (16 * NB), p = (i - u * 16 * NB) >> 4, g = (i >> 2) & 3, q = i & 3;
        const int r0 = 16 * (unit0 + u) + 4 * g - slot0;  // the first of the item's 4 tokens
        if (r0 + 4 <= 0 || r0 >= n) continue;
        const bool all = r0 >= 0 && r0 + 4 <= n;
        float x[4][2][4];  // token, 16 dims, dim
#pragma unroll
        for (int e = 0; e < 4; e++)
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const int d = 32 * p + 16 * t + 4 * q;
                if (d < hd && r0 + e >= 0 && r0 + e < n) {
                    load_n<ACT>(src, (int64_t)(row0 + r0 + e) * ld + (int64_t)h * hd + d, x[e][t]);
                } else {
#pragma unroll
                    for (int k = 0; k < 4; k++) x[e][t][k] = 0.0f;
                }
            }
        int apart;
        const int64_t at = (int64_t)(unit0 + u) * 16 * hdp + v_item<I8>(hdp, p, g, q, apart);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            using Code = std::conditional_t<I8, uint8_t, _Float16>;
            Code w[8];
#pragma unroll
            for (int f = 0; f < 8; f++) {
                if constexpr (I8) w[f] = (uint8_t)code_of(x[f & 3][f >> 2][k], inv);
                else w[f] = (_Float16)x[f & 3][f >> 2][k];
            }
            Code *o = reinterpret_cast<Code *>(a.v) + base + at + k * apart;
            if (all) {
                __builtin_memcpy(__builtin_assume_aligned(o, 8 * sizeof(Code)), w, 8 * sizeof(Code));
            } else {
#pragma unroll
                for (int f = 0; f < 8; f++)
                    if (r0 + (f & 3) >= 0 && r0 + (f & 3) < n) o[f] = w[f];
            }
        }
    }
}

// units of 16 tokens that a sequence's rows reach
__device__ __forceinline__ int units_touched(const Seq &s) {
    return s.cnt > 0 ? (((s.len0 & 15) + s.cnt - 1) >> 4) + 1 : 0;
}

// One block: one unit of 16 tokens, its K/V heads' items in turn, or a share of
// them where there are few units.  8 bits to bf16, 8176 tokens of 8 heads of 128:
// 13.7 us, 3.7 TB/s.
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
