// Log probabilities of rows of logits (lcmoe_logprobs_dev): for a row x,
//   m = max x,  Z = sum e^(x - m),  T = sum (x - m) e^(x - m),
//   log p(t) = x_t - m - log Z,  entropy = log Z - T / Z,
// and the n largest logits.  Several blocks may share a row: each leaves its
// (m, Z, T) and its n largest, which k_logprobs_join brings together.
//
// The n largest: a thread keeps the largest of its own elements; the n-th
// largest of the threads' is a bound that n elements at least reach, and that
// no element of any other thread does.  So only n threads' elements are looked
// at again, and their survivors ranked.  Keys are (logit, lower index first),
// so no two are equal and the result does not depend on any order.

#include "kv_device.h"

namespace lcmoe {
namespace {

constexpr int kThreads = 256;
constexpr int kTopMost = 32;
constexpr int kPerThread = 128;                 // elements of one thread, at most
constexpr int kSpan = kThreads * kPerThread;    // elements of one block, at most
constexpr int kSurvivors = kTopMost * kPerThread;

// larger for the larger logit, then for the lower index; NaN as -inf.  Zero is
// below every element's key.
__device__ __forceinline__ uint64_t key_of(float x, int i) {
    x = x == x ? x + 0.0f : -INFINITY;  // -0 + 0 = +0: equal to it
    uint32_t u = __float_as_uint(x);
    u ^= (uint32_t)((int32_t)u >> 31) | 0x80000000u;
    return ((uint64_t)u << 32) | (uint32_t)~i;
}
__device__ __forceinline__ int key_index(uint64_t k) { return (int)~(uint32_t)k; }
__device__ __forceinline__ float key_value(uint64_t k) {
    const uint32_t u = (uint32_t)(k >> 32);
    return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}

template <int TYPE>
__device__ __forceinline__ float load1(const void *x, int64_t e) {
    if constexpr (TYPE == LCMOE_TYPE_F32) return static_cast<const float *>(x)[e];
    else if constexpr (TYPE == LCMOE_TYPE_F16) return dh2f(static_cast<const uint16_t *>(x)[e]);
    else return __uint_as_float((uint32_t)static_cast<const uint16_t *>(x)[e] << 16);
}

struct Stat {
    float m, z, t;  // max, sum e^(x - m), sum (x - m) e^(x - m)
};
constexpr float kLog2e = 1.44269504088896340736f;

// s in units of e^m, m >= s.m
__device__ __forceinline__ void rebase(Stat &s, float m) {
    if (s.m == m || s.m == -INFINITY) {  // an empty sum, or NaN and -inf alone
        s.m = m;
        return;
    }
    const float d = s.m - m, f = __builtin_amdgcn_exp2f(d * kLog2e);
    s.t = f > 0.0f || f != f ? f * (s.t + d * s.z) : 0.0f;
    s.z *= f;
    s.m = m;
}
__device__ __forceinline__ void join(Stat &s, Stat o) {
    const float m = fmaxf(s.m, o.m);
    rebase(s, m);
    rebase(o, m);
    s.z += o.z;
    s.t += o.t;
}
__device__ __forceinline__ void add(Stat &s, float x) {  // x <= s.m
    if (x == -INFINITY) return;
    const float d = x - s.m, e = __builtin_amdgcn_exp2f(d * kLog2e);
    s.z += e;
    if (e != 0.0f) s.t = __builtin_fmaf(d, e, s.t);
}
__device__ __forceinline__ Stat wave_join(Stat s) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const Stat u = {__shfl_xor(s.m, o, 64), __shfl_xor(s.z, o, 64), __shfl_xor(s.t, o, 64)};
        join(s, u);
    }
    return s;
}

// the results of a finished row
template <int TYPE>
__device__ void finish(const Stat &s, const void *x, int64_t row, int64_t ld, int vocab,
                       const int32_t *given, int n_given, float *given_lp, float *entropy, int top,
                       const uint64_t *keys, int32_t *top_id, float *top_lp) {
    // a row without a logit above -inf: -inf for every token, no entropy
    const bool empty = s.m == -INFINITY && s.z == 0.0f;
    const float lz = logf(s.z);
    const auto lp = [&](float v) { return empty ? -INFINITY : v - s.m - lz; };
    for (int i = threadIdx.x; i < n_given; i += blockDim.x) {
        const int id = given[row * n_given + i];
        given_lp[row * n_given + i] =
            id >= 0 && id < vocab ? lp(load1<TYPE>(x, row * ld + id)) : 0.0f;
    }
    if (entropy && threadIdx.x == 0) entropy[row] = empty ? 0.0f : lz - s.t / s.z;
    for (int i = threadIdx.x; i < top; i += blockDim.x) {
        top_id[row * top + i] = keys[i] ? key_index(keys[i]) : -1;
        top_lp[row * top + i] = keys[i] ? lp(key_value(keys[i])) : -INFINITY;
    }
}

template <int TYPE, bool TOP>
__global__ __launch_bounds__(kThreads) void k_logprobs(const void *__restrict__ x, int64_t ld,
                                                       int vocab, int span,
                                                       const int32_t *__restrict__ given,
                                                       int n_given, float *__restrict__ given_lp,
                                                       float *__restrict__ entropy, int top,
                                                       int32_t *__restrict__ top_id,
                                                       float *__restrict__ top_lp,
                                                       Stat *__restrict__ part,
                                                       uint64_t *__restrict__ part_key) {
    const int64_t row = blockIdx.y;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int i0 = blockIdx.x * span, i1 = min(vocab, i0 + span);
    Stat s = {-INFINITY, 0.0f, 0.0f};
    uint64_t best = 0;
    for (int i = i0 + tid; i < i1; i += kThreads) {
        const float v = load1<TYPE>(x, row * ld + i);
        if (v > s.m) rebase(s, v);
        add(s, v);
        if constexpr (TOP) {
            const uint64_t k = key_of(v, i);
            if (k > best) best = k;
        }
    }
    __shared__ Stat s_stat[kThreads / 64];
    s = wave_join(s);
    if (lane == 0) s_stat[wave] = s;
    __shared__ uint64_t s_max[kThreads];
    __shared__ uint64_t s_top[kTopMost];
    if constexpr (TOP) s_max[tid] = best;
    __syncthreads();
    s = s_stat[0];
#pragma unroll
    for (int w = 1; w < kThreads / 64; w++) join(s, s_stat[w]);
    if constexpr (TOP) {
        __shared__ uint64_t s_key[kSurvivors];
        __shared__ int s_who[kTopMost], s_n;
        // the threads with the n largest maxima, and the n-th of those
        int rank = 0;
        for (int j = 0; j < kThreads; j++) rank += s_max[j] > best;
        if (tid < kTopMost) s_top[tid] = 0;
        if (tid == 0) s_n = 0;
        __syncthreads();
        if (best && rank < top) {
            s_who[rank] = tid;
            s_top[rank] = best;
        }
        __syncthreads();
        const uint64_t bound = s_top[top - 1];  // 0: fewer than n threads have any
        for (int w = 0; w < top; w++) {
            if (!s_top[w]) break;
            for (int i = i0 + s_who[w] + kThreads * tid; i < i1; i += kThreads * kThreads) {
                const uint64_t k = key_of(load1<TYPE>(x, row * ld + i), i);
                if (k >= bound) s_key[atomicAdd(&s_n, 1)] = k;
            }
        }
        __syncthreads();
        const int n = s_n;
        if (tid < kTopMost) s_top[tid] = 0;
        __syncthreads();
        for (int i = tid; i < n; i += kThreads) {
            const uint64_t k = s_key[i];
            int r = 0;
            for (int j = 0; j < n; j++) r += s_key[j] > k;
            if (r < top) s_top[r] = k;
        }
        __syncthreads();
    }
    if (gridDim.x == 1) {
        finish<TYPE>(s, x, row, ld, vocab, given, n_given, given_lp, entropy, top, s_top, top_id,
                     top_lp);
        return;
    }
    const int64_t at = row * gridDim.x + blockIdx.x;
    if (tid == 0) part[at] = s;
    if constexpr (TOP)
        for (int i = tid; i < top; i += kThreads) part_key[at * top + i] = s_top[i];
}

// One wave per row: the statistics of `parts` blocks, and the n largest of
// their ordered lists, one at a time by their heads.
template <int TYPE>
__global__ __launch_bounds__(64) void k_logprobs_join(const void *__restrict__ x, int64_t ld,
                                                      int vocab, int parts,
                                                      const int32_t *__restrict__ given,
                                                      int n_given, float *__restrict__ given_lp,
                                                      float *__restrict__ entropy, int top,
                                                      int32_t *__restrict__ top_id,
                                                      float *__restrict__ top_lp,
                                                      const Stat *__restrict__ part,
                                                      const uint64_t *__restrict__ part_key) {
    __shared__ uint64_t s_top[kTopMost];
    const int64_t row = blockIdx.x;
    const int lane = threadIdx.x;
    Stat s = {-INFINITY, 0.0f, 0.0f};
    for (int p = lane; p < parts; p += 64) join(s, part[row * parts + p]);
    s = wave_join(s);
    uint64_t last = ~(uint64_t)0;
    for (int i = 0; i < top; i++) {
        uint64_t best = 0;
        for (int p = lane; p < parts; p += 64) {
            const uint64_t *k = part_key + (row * parts + p) * top;
            int f = 0;
            while (f < top && k[f] >= last) f++;
            if (f < top && k[f] > best) best = k[f];
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const uint64_t u = __shfl_xor(best, o, 64);
            if (u > best) best = u;
        }
        if (lane == 0) s_top[i] = best;
        last = best;
    }
    __syncthreads();
    finish<TYPE>(s, x, row, ld, vocab, given, n_given, given_lp, entropy, top, s_top, top_id, top_lp);
}

// elements of a row that one block takes
int span_of(int rows, int vocab) {
    int parts = (vocab + kSpan - 1) / kSpan;
    while ((int64_t)rows * parts < 1024 && vocab / (2 * parts) >= 4 * kThreads) parts *= 2;
    return (vocab + parts - 1) / parts;
}

}  // namespace

int64_t logprobs_bytes(int type, int rows, int vocab, int top) {
    const int span = span_of(rows, vocab), parts = (vocab + span - 1) / span;
    return parts == 1 ? 0 : (int64_t)rows * parts * (16 + 8 * (int64_t)top);
}

hipError_t launch_logprobs(int type, const void *x, int64_t ld, int rows, int vocab,
                           const int32_t *given, int n_given, float *given_lp, float *entropy,
                           int top, int32_t *top_id, float *top_lp, void *ws, hipStream_t st) {
    const int span = span_of(rows, vocab), parts = (vocab + span - 1) / span;
    uint64_t *keys = static_cast<uint64_t *>(ws);
    Stat *part = reinterpret_cast<Stat *>(keys + (parts == 1 ? 0 : (int64_t)rows * parts * top));
    const auto go = [&](auto type_c) {
        constexpr int TYPE = decltype(type_c)::value;
        // grid.y holds 65535 rows; more run in turns
        for (int64_t r0 = 0; r0 < rows; r0 += 65535) {
            const unsigned n = (unsigned)std::min<int64_t>(65535, rows - r0);
            const void *xr = static_cast<const uint8_t *>(x) +
                             r0 * ld * (TYPE == LCMOE_TYPE_F32 ? 4 : 2);
            const int32_t *g = given ? given + r0 * n_given : nullptr;
            float *glp = given_lp ? given_lp + r0 * n_given : nullptr;
            float *ent = entropy ? entropy + r0 : nullptr;
            int32_t *tid = top_id ? top_id + r0 * top : nullptr;
            float *tlp = top_lp ? top_lp + r0 * top : nullptr;
            auto *kern = top ? k_logprobs<TYPE, true> : k_logprobs<TYPE, false>;
            hipLaunchKernelGGL(kern, dim3(parts, n), dim3(kThreads), 0, st, xr, ld, vocab, span, g,
                               n_given, glp, ent, top, tid, tlp, part + r0 * parts,
                               keys + r0 * parts * top);
            if (parts > 1)
                hipLaunchKernelGGL(k_logprobs_join<TYPE>, dim3(n), dim3(64), 0, st, xr, ld, vocab,
                                   parts, g, n_given, glp, ent, top, tid, tlp, part + r0 * parts,
                                   keys + r0 * parts * top);
            if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        }
        return hipSuccess;
    };
    switch (type) {
    case LCMOE_TYPE_F32: return go(std::integral_constant<int, LCMOE_TYPE_F32>());
    case LCMOE_TYPE_F16: return go(std::integral_constant<int, LCMOE_TYPE_F16>());
    default: return go(std::integral_constant<int, LCMOE_TYPE_BF16>());
    }
}

}  // namespace lcmoe
