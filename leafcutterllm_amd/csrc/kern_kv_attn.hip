// Causal attention of a ragged batch over a paged cache
// (lcmoe_kv_attention_dev).  The layout is in kv_device.h.

#include "kv_device.h"

namespace lcmoe {
namespace {

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}

// One wave: one row, one head; 64 keys at a time.
template <int ACT, bool I8>
__global__ __launch_bounds__(64) void k_kv_attn(KvArgs a, const void *__restrict__ q, int64_t ldq,
                                                const float *__restrict__ rope, float scale,
                                                void *__restrict__ out, int64_t ldo) {
    __shared__ float s_q[256], s_p[64];
    const int lane = threadIdx.x, hh = blockIdx.y, hd = a.hd, half = hd / 2;
    int i = 0;
    const int b = find_tile(a, blockIdx.x, [](const Seq &s) { return max(s.cnt, 0); }, i);
    if (b < 0) return;
    const Seq s = sequence(a, b);
    const int h = hh / (a.H / a.KVH), pos = s.len0 + i, P = 1 << a.plog;
    const auto load = [&](int d) {
        const int64_t e = (int64_t)(s.row0 + i) * ldq + (int64_t)hh * hd + d;
        if constexpr (ACT == LCMOE_TYPE_F32) return static_cast<const float *>(q)[e];
        else if constexpr (ACT == LCMOE_TYPE_F16) return dh2f(static_cast<const uint16_t *>(q)[e]);
        else return __uint_as_float((uint32_t)static_cast<const uint16_t *>(q)[e] << 16);
    };
    for (int d = lane; d < half; d += 64) {
        const float x = load(d), z = load(d + half);
        if (rope) {
            const float *cs = rope + ((int64_t)(a.rope_abs ? pos : i) * half + d) * 2;
            s_q[d] = x * cs[0] - z * cs[1];
            s_q[d + half] = x * cs[1] + z * cs[0];
        } else {
            s_q[d] = x;
            s_q[d + half] = z;
        }
    }
    __syncthreads();
    float m = -INFINITY, l = 0.0f, acc[4] = {0, 0, 0, 0};
    for (int p0 = 0; p0 <= pos; p0 += 64) {
        const int p = p0 + lane;
        const int page = p <= pos ? a.pages[(int64_t)b * a.max_pages + (p >> a.plog)] : -1;
        float x = -INFINITY;
        if (page >= 0 && page < a.n_pages) {
            const int64_t u = unit_base(a, page, h, (p & (P - 1)) >> 4);
            float dot = 0.0f;
            for (int d = 0; d < hd; d++) {
                const int64_t at = u + k_place<I8>(a.hdp, p & 15, d);
                const float k = I8 ? (float)(int8_t)a.k[at]
                                   : (float)reinterpret_cast<const _Float16 *>(a.k)[at];
                dot = __builtin_fmaf(s_q[d], k, dot);
            }
            if (I8) dot *= a.scale[((int64_t)page * a.KVH + h) * 2];
            x = dot * scale;
        }
        const float mn = fmaxf(m, wave_max(x));
        const float base = mn == -INFINITY ? 0.0f : mn;
        const float keep = expf(m - base), e = expf(x - base);
        s_p[lane] = e;
        l = l * keep + wave_sum(e);
#pragma unroll
        for (int c = 0; c < 4; c++) acc[c] *= keep;
        m = mn;
        __syncthreads();
        for (int t = 0; t < min(64, pos + 1 - p0); t++) {
            const int pt = p0 + t, pg = a.pages[(int64_t)b * a.max_pages + (pt >> a.plog)];
            if (pg < 0 || pg >= a.n_pages) continue;
            const int64_t u = unit_base(a, pg, h, (pt & (P - 1)) >> 4);
            const float w = I8 ? s_p[t] * a.scale[((int64_t)pg * a.KVH + h) * 2 + 1] : s_p[t];
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int d = lane + 64 * c;
                if (d >= hd) break;
                const int64_t at = u + v_place<I8>(a.hdp, pt & 15, d);
                const float v = I8 ? (float)(int8_t)a.v[at]
                                   : (float)reinterpret_cast<const _Float16 *>(a.v)[at];
                acc[c] = __builtin_fmaf(w, v, acc[c]);
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int c = 0; c < 4; c++) {
        const int d = lane + 64 * c;
        if (d < hd)
            store1<ACT>(out, (int64_t)(s.row0 + i) * ldo + (int64_t)hh * hd + d,
                        l == 0.0f ? 0.0f : acc[c] / l);
    }
}

}  // namespace

int64_t kv_attention_floats(const KvArgs &) { return 0; }

hipError_t launch_kv_attention(const KvArgs &a, const void *q, int64_t ldq, const float *rope,
                               float scale, void *out, int64_t ldo, bool vec, float *ws,
                               hipStream_t st) {
    const dim3 grid(a.n_rows, a.H);
    const auto go = [&](auto kern) {
        hipLaunchKernelGGL(kern, grid, dim3(64), 0, st, a, q, ldq, rope, scale, out, ldo);
        return hipGetLastError();
    };
    if (a.act == LCMOE_TYPE_F32)
        return a.i8 ? go(k_kv_attn<LCMOE_TYPE_F32, true>) : go(k_kv_attn<LCMOE_TYPE_F32, false>);
    if (a.act == LCMOE_TYPE_F16)
        return a.i8 ? go(k_kv_attn<LCMOE_TYPE_F16, true>) : go(k_kv_attn<LCMOE_TYPE_F16, false>);
    return a.i8 ? go(k_kv_attn<LCMOE_TYPE_BF16, true>) : go(k_kv_attn<LCMOE_TYPE_BF16, false>);
}

}  // namespace lcmoe
