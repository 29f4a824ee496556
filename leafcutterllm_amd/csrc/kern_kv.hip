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

// y = the key's dims c .. c + 7 and h + c .. h + c + 7 (h = head_dim / 2),
// rotated by (cos, sin) = rope[c .. c + 7]:
//   y[d] = x[d] cos - x[h + d] sin,  y[h + d] = x[d] sin + x[h + d] cos.
// Products of two f32 are exact in 64 bits.
template <int ACT>
__device__ __forceinline__ void rotated8(const void *src, int64_t e, int h, bool vec,
                                         const float *cs, double (&lo)[8], double (&hi)[8]) {
    float x[8], z[8];
    load8<ACT>(src, e, vec, x);
    load8<ACT>(src, e + h, vec, z);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const double c = cs ? (double)cs[2 * i] : 1.0, s = cs ? (double)cs[2 * i + 1] : 0.0;
        lo[i] = cs ? x[i] * c - z[i] * s : x[i];
        hi[i] = cs ? x[i] * s + z[i] * c : z[i];
    }
}

// One block: the new tokens of one page, one K/V head, keys (z = 0) or values
// (z = 1).  In 8 bits the page's scale S' = max(S, max |new| / 127), S = 0
// where the page's first token is new; codes that were there are moved to the
// new scale where it grew; the new ones follow.  One block owns a page's head,
// so nothing here depends on the order in which blocks run.
template <int ACT, bool I8>
__global__ __launch_bounds__(256) void k_kv_append(KvArgs a, const void *__restrict__ ksrc,
                                                   int64_t ldk, const void *__restrict__ vsrc,
                                                   int64_t ldv, const float *__restrict__ rope,
                                                   bool vec) {
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
    const auto key8 = [&](int i, double (&lo)[8], double (&hi)[8]) {
        const int t = i / KC, c = 8 * (i % KC);
        const int rot = a.rope_abs ? s.len0 + t0 + t : t0 + t;
        rotated8<ACT>(src, (int64_t)(row0 + t) * ld + (int64_t)h * hd + c, half, vec,
                      rope ? rope + ((int64_t)rot * half + c) * 2 : nullptr, lo, hi);
    };
    double inv = 0.0;
    if constexpr (I8) {
        double most = 0.0;
        const auto larger = [&](double y) {
            const double m = fabs(y);
            if (m > most && m < INFINITY) most = m;
        };
        if (!value) {
            for (int i = tid; i < n * KC; i += 256) {
                double lo[8], hi[8];
                key8(i, lo, hi);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    larger(lo[e]);
                    larger(hi[e]);
                }
            }
        } else {
            const int C = hd / 8;
            for (int i = tid; i < n * C; i += 256) {
                float x[8];
                load8<ACT>(src, (int64_t)(row0 + i / C) * ld + (int64_t)h * hd + 8 * (i % C), vec, x);
#pragma unroll
                for (int e = 0; e < 8; e++) larger(x[e]);
            }
        }
        __shared__ double s_most[4];
        most = wave_max(most);
        if ((tid & 63) == 0) s_most[tid >> 6] = most;
        __syncthreads();
        most = fmax(fmax(s_most[0], s_most[1]), fmax(s_most[2], s_most[3]));
        float *sp = a.scale + ((int64_t)page * a.KVH + h) * 2 + value;
        const float old = slot0 ? *sp : 0.0f;
        const float scale = fmaxf(old, (float)(most / 127.0));
        inv = scale > 0.0f ? 1.0 / (double)scale : 0.0;
        if (slot0 && scale > old) {
            const double ratio = (double)old / (double)scale;
            const auto moved = [&](uint32_t w) {
                uint32_t o = 0;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int q = (int)__builtin_rint((double)(int8_t)(w >> 8 * e) * ratio);
                    o |= (uint32_t)(uint8_t)q << 8 * e;
                }
                return o;
            };
            if (!value) {
                for (int i = tid; i < slot0 * (hdp / 8); i += 256) {
                    const int slot = i / (hdp / 8), d = 8 * (i % (hdp / 8));
                    uintx2 *p = reinterpret_cast<uintx2 *>(p8 + (int64_t)(slot >> 4) * 16 * hdp +
                                                           k_place<true>(hdp, slot & 15, d));
                    const uintx2 w = *p;
                    *p = uintx2{moved(w[0]), moved(w[1])};
                }
            } else {
                for (int i = tid; i < (slot0 + 3) / 4 * hd; i += 256) {
                    const int slot = 4 * (i / hd), d = i % hd;
                    uint32_t *p = reinterpret_cast<uint32_t *>(p8 + (int64_t)(slot >> 4) * 16 * hdp +
                                                               v_place<true>(hdp, slot & 15, d));
                    *p = moved(*p);
                }
            }
        }
        __syncthreads();  // *sp read by every thread, the moved codes written
        if (tid == 0) *sp = scale;
    }
    if (!value) {
        for (int i = tid; i < n * KC; i += 256) {
            double lo[8], hi[8];
            key8(i, lo, hi);
            const int slot = slot0 + i / KC, c = 8 * (i % KC);
            const int64_t u = (int64_t)(slot >> 4) * 16 * hdp;
            if constexpr (I8) {
                uintx2 wl = {0, 0}, wh = {0, 0};
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    wl[e >> 2] |= (uint32_t)(uint8_t)code_of(lo[e], inv) << 8 * (e & 3);
                    wh[e >> 2] |= (uint32_t)(uint8_t)code_of(hi[e], inv) << 8 * (e & 3);
                }
                *reinterpret_cast<uintx2 *>(p8 + u + k_place<true>(hdp, slot & 15, c)) = wl;
                *reinterpret_cast<uintx2 *>(p8 + u + k_place<true>(hdp, slot & 15, half + c)) = wh;
            } else {
                half8 wl, wh;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    wl[e] = (_Float16)lo[e];
                    wh[e] = (_Float16)hi[e];
                }
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
    // values: four tokens of eight dims, whose places are contiguous per dim
    const int C = hd / 8, q0 = slot0 >> 2, nq = ((slot0 + n + 3) >> 2) - q0;
    for (int i = tid; i < nq * C; i += 256) {
        const int slot = 4 * (q0 + i / C), d = 8 * (i % C);
        float x[4][8];
        bool mine[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            mine[e] = slot + e >= slot0 && slot + e < slot0 + n;
            if (mine[e])
                load8<ACT>(src, (int64_t)(row0 + slot + e - slot0) * ld + (int64_t)h * hd + d, vec,
                           x[e]);
        }
        const bool all = mine[0] && mine[3];
        const int64_t u = (int64_t)(slot >> 4) * 16 * hdp;
#pragma unroll
        for (int f = 0; f < 8; f++) {
            const int64_t at = u + v_place<I8>(hdp, slot & 15, d + f);
            if constexpr (I8) {
                uint32_t w = 0;
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (mine[e]) w |= (uint32_t)(uint8_t)code_of(x[e][f], inv) << 8 * e;
                if (all) {
                    *reinterpret_cast<uint32_t *>(p8 + at) = w;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (mine[e]) p8[at + e] = (uint8_t)(w >> 8 * e);
                }
            } else {
                if (all) {
                    *reinterpret_cast<half4 *>(p16 + at) =
                        half4{(_Float16)x[0][f], (_Float16)x[1][f], (_Float16)x[2][f],
                              (_Float16)x[3][f]};
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (mine[e]) p16[at + e] = (_Float16)x[e][f];
                }
            }
        }
    }
}

// units of 16 tokens that a sequence's rows reach
__device__ __forceinline__ int units_touched(const Seq &s) {
    return s.cnt > 0 ? (((s.len0 & 15) + s.cnt - 1) >> 4) + 1 : 0;
}

// One block: one unit of 16 tokens, one K/V head.
template <int ACT, bool I8>
__global__ __launch_bounds__(256) void k_kv_read(KvArgs a, void *__restrict__ ko, int64_t ldk,
                                                 void *__restrict__ vo, int64_t ldv, bool vec) {
    const int h = blockIdx.y, tid = threadIdx.x;
    int j = 0;
    const int b = find_tile(a, blockIdx.x, [&](const Seq &s) { return units_touched(s); }, j);
    if (b < 0) return;
    const Seq s = sequence(a, b);
    const int p0 = ((s.len0 >> 4) + j) << 4;  // the unit's first position
    const int page = a.pages[(int64_t)b * a.max_pages + (p0 >> a.plog)];
    const bool held = page >= 0 && page < a.n_pages;
    const int64_t u = unit_base(a, held ? page : 0, h, (p0 & ((1 << a.plog) - 1)) >> 4);
    float sk = 1.0f, sv = 1.0f;
    if (I8 && held) {
        sk = a.scale[((int64_t)page * a.KVH + h) * 2];
        sv = a.scale[((int64_t)page * a.KVH + h) * 2 + 1];
    }
    const int hd = a.hd, C = hd / 8;
    const auto value = [&](const uint8_t *pool, int64_t at, float scale) {
        if (!held) return 0.0f;
        if constexpr (I8) return (float)(int8_t)pool[at] * scale;
        else return (float)reinterpret_cast<const _Float16 *>(pool)[at];
    };
    for (int i = tid; i < 16 * C; i += 256) {
        const int r = i / C, d = 8 * (i % C), t = p0 + r - s.len0;
        if (t < 0 || t >= s.cnt) continue;
        float k[8], v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            k[e] = value(a.k, u + k_place<I8>(a.hdp, r, d + e), sk);
            v[e] = value(a.v, u + v_place<I8>(a.hdp, r, d + e), sv);
        }
        store8<ACT>(ko, (int64_t)(s.row0 + t) * ldk + (int64_t)h * hd + d, vec, k);
        store8<ACT>(vo, (int64_t)(s.row0 + t) * ldv + (int64_t)h * hd + d, vec, v);
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
                            const float *rope, bool vec, hipStream_t st) {
    const dim3 grid((unsigned)most_blocks(a, 1 << a.plog), a.KVH, 2);
    return by_type(a.act, a.i8, [&](auto act, auto i8) {
        hipLaunchKernelGGL((k_kv_append<decltype(act)::value, decltype(i8)::value>), grid, dim3(256),
                           0, st, a, k, ldk, v, ldv, rope, vec);
        return hipGetLastError();
    });
}

hipError_t launch_kv_read(const KvArgs &a, void *k, int64_t ldk, void *v, int64_t ldv, bool vec,
                          hipStream_t st) {
    const dim3 grid((unsigned)most_blocks(a, 16), a.KVH);
    return by_type(a.act, a.i8, [&](auto act, auto i8) {
        hipLaunchKernelGGL((k_kv_read<decltype(act)::value, decltype(i8)::value>), grid, dim3(256),
                           0, st, a, k, ldk, v, ldv, vec);
        return hipGetLastError();
    });
}

}  // namespace lcmoe
