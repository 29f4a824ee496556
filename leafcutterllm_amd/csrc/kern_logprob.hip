// Log probabilities of rows of logits (lcmoe_logprobs_dev): for a row x,
//   m = max x,  Z = sum e^(x - m),  T = sum (x - m) e^(x - m),
//   log p(t) = x_t - m - log Z,  entropy = log Z - T / Z,
// and the n largest logits.  Several blocks may share a row: each leaves its
// (m, Z, T) and its n largest, which k_logprobs_join brings together.
//
// The n largest: a thread keeps its elements in registers.  Lane l of all waves
// has a largest one; the n-th of those 64 is a bound that n elements at least
// reach, and few more (of equally spread ones 64 log(64 / (64 - n)) are
// expected: 24 for 20).  They go to a list in LDS and are ranked there.  Keys
// are (logit, lower index first), so no two are equal and the result does not
// depend on any order.  A row made so that the list overflows is gone through n
// times instead.

#include "kv_device.h"

namespace lcmoe {
namespace {

constexpr int kTopMost = 32;
constexpr int kList = 1024;  // what reaches the bound, at most
constexpr int kRegs = 32;    // elements of a thread
constexpr int kFew = 128;    // keys that a join ranks without a bound

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

// V = 16 bytes' worth of elements from i on, -inf if they pass `end`; rows
// need be aligned to their elements only
template <int TYPE> constexpr int kVec = TYPE == LCMOE_TYPE_F32 ? 4 : 8;
template <int TYPE>
__device__ __forceinline__ void load_vec(const void *x, int64_t row, int i, int end, float *o) {
    constexpr int V = kVec<TYPE>;
    if (i + V <= end) {
        uintx4 w;
        __builtin_memcpy(&w, static_cast<const uint8_t *>(x) + (row + i) * (16 / V), 16);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if constexpr (TYPE == LCMOE_TYPE_F32) {
                o[k] = __uint_as_float(w[k]);
            } else if constexpr (TYPE == LCMOE_TYPE_F16) {
                o[2 * k] = dh2f(w[k] & 0xffff);
                o[2 * k + 1] = dh2f(w[k] >> 16);
            } else {
                o[2 * k] = __uint_as_float(w[k] << 16);
                o[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < V; k++) o[k] = -INFINITY;
    }
}
// what is left of a span behind its last 16 bytes: an element for each of the
// first few threads
template <int TYPE>
__device__ __forceinline__ float load_tail(const void *x, int64_t row, int i0, int i1, int &at) {
    const int rem = (i1 - i0) % kVec<TYPE>;
    at = i1 - rem + threadIdx.x;
    return at < i1 ? load1<TYPE>(x, row + at) : -INFINITY;
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
// N elements, -inf where there is none
template <int N>
__device__ __forceinline__ void add(Stat &s, const float (&x)[N]) {
    float m = s.m;
#pragma unroll
    for (int i = 0; i < N; i++) m = fmaxf(m, x[i]);
    rebase(s, m);
    const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const float d = x[i] - base, e = __builtin_amdgcn_exp2f(d * kLog2e);
        s.z += e;
        s.t = __builtin_fmaf(e != 0.0f ? d : 0.0f, e, s.t);
    }
}
template <int N>
__device__ __forceinline__ Stat wave_join(Stat s) {
#pragma unroll 1
    for (int o = N / 2; o > 0; o >>= 1) {
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

// the block's statistics, in every thread; s_stat: one a wave
template <int T>
__device__ __forceinline__ Stat block_join(Stat s, Stat *s_stat) {
    s = wave_join<64>(s);
    if ((threadIdx.x & 63) == 0) s_stat[threadIdx.x >> 6] = s;
    __syncthreads();
    return wave_join<T / 64>(s_stat[threadIdx.x & (T / 64 - 1)]);
}

struct RowArgs {
    const void *x;
    int64_t ld;
    int vocab, span;  // elements of a row, of a block
    const int32_t *given;
    int n_given;
    float *given_lp, *entropy;
    int top;
    int32_t *top_id;
    float *top_lp;
    Stat *part;
    uint64_t *part_key;
};

template <int TYPE>
__device__ __forceinline__ void finish(const RowArgs &a, const Stat &s, int64_t row, const uint64_t *keys) {
    finish<TYPE>(s, a.x, row, a.ld, a.vocab, a.given, a.n_given, a.given_lp, a.entropy, a.top, keys,
                 a.top_id, a.top_lp);
}

// Statistics alone: a block goes through its span with 32 elements a thread in
// flight.
template <int TYPE>
__global__ __launch_bounds__(256) void k_logprobs(RowArgs a) {
    constexpr int T = 256, V = kVec<TYPE>;
    __shared__ Stat s_stat[T / 64];
    const int64_t row = blockIdx.y;
    const int i0 = blockIdx.x * a.span, i1 = min(a.vocab, i0 + a.span);
    Stat s = {-INFINITY, 0.0f, 0.0f};
    for (int i = i0 + V * threadIdx.x; i < i1; i += T * kRegs) {
        float x[kRegs];
#pragma unroll
        for (int k = 0; k < kRegs / V; k++) load_vec<TYPE>(a.x, row * a.ld, i + k * T * V, i1, x + k * V);
        add(s, x);
    }
    int at;
    const float xt[1] = {load_tail<TYPE>(a.x, row * a.ld, i0, i1, at)};
    add(s, xt);
    s = block_join<T>(s, s_stat);
    if (gridDim.x == 1) finish<TYPE>(a, s, row, nullptr);
    else if (threadIdx.x == 0) a.part[row * gridDim.x + blockIdx.x] = s;
}

// The largest of the keys below `last`, of the whole block.
template <int T>
__device__ __forceinline__ uint64_t block_max(uint64_t k, uint64_t *s_red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint64_t u = __shfl_xor(k, o, 64);
        if (u > k) k = u;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s_red[threadIdx.x >> 6] = k;
    __syncthreads();
    k = s_red[0];
    for (int w = 1; w < T / 64; w++)
        if (s_red[w] > k) k = s_red[w];
    return k;
}

// how many lanes' u are above k
__device__ __forceinline__ int lanes_above(uint64_t u, uint64_t k) {
    const uint32_t lo = (uint32_t)u, hi = (uint32_t)(u >> 32);
    int n = 0;
#pragma unroll 8
    for (int j = 0; j < 64; j++)
        n += ((uint32_t)__builtin_amdgcn_readlane(lo, j) |
              (uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, j) << 32) > k;
    return n;
}
// of the wave's keys (one a lane, 0 for none) the n-th largest
__device__ __forceinline__ uint64_t wave_nth(uint64_t k, int n) {
    const uint64_t at = __ballot(k != 0 && lanes_above(k, k) == n - 1);
    return at ? __shfl(k, __builtin_ctzll(at), 64) : 0;
}
// s_top = the `top` largest of n keys in LDS (others 0), largest first; a wave
// ranks 64 keys
template <int T>
__device__ __forceinline__ void rank_list(const uint64_t *s_key, int n, int top, uint64_t *s_top) {
    if (threadIdx.x < kTopMost) s_top[threadIdx.x] = 0;
    __syncthreads();
#pragma unroll 1
    for (int i = threadIdx.x; i < ((n + 63) & ~63); i += T) {
        const uint64_t k = i < n ? s_key[i] : 0;
        int r = 0;
#pragma unroll 1
        for (int j = threadIdx.x & 63; j < ((n + 63) & ~63); j += 64)
            r += lanes_above(j < n ? s_key[j] : 0, k);
        if (i < n && r < top) s_top[r] = k;
    }
    __syncthreads();
}

// Statistics and the n largest of up to 32 T elements.
template <int TYPE, int T>
__global__ __launch_bounds__(T) void k_logprobs_top(RowArgs a) {
    constexpr int V = kVec<TYPE>;
    __shared__ Stat s_stat[T / 64];
    __shared__ uint64_t s_red[T / 64], s_top[kTopMost], s_key[kList];
    __shared__ uint64_t s_bound;
    __shared__ int s_n;
    const int64_t row = blockIdx.y;
    const int i0 = blockIdx.x * a.span, i1 = min(a.vocab, i0 + a.span), tid = threadIdx.x;
    const int64_t x0 = row * a.ld;
    const auto index = [&](int e) { return i0 + V * (tid + e / V * T) + e % V; };
    float x[kRegs];
#pragma unroll
    for (int k = 0; k < kRegs / V; k++) load_vec<TYPE>(a.x, x0, index(k * V), i1, x + k * V);
    int tail_at;
    const float xt[1] = {load_tail<TYPE>(a.x, x0, i0, i1, tail_at)};
    // the key of the lane's largest, 0 if it has none; NaN counts as -inf
    float best = x[0];
#pragma unroll
    for (int e = 1; e < kRegs; e++) best = fmaxf(best, x[e]);
    uint32_t hit = 0;
#pragma unroll
    for (int e = kRegs - 1; e >= 0; e--) hit = 2 * hit + (x[e] == best);
    const int at = best > -INFINITY ? index(__builtin_ctz(hit)) : index(0);
    uint64_t own = at + (best > -INFINITY ? 0 : V - 1) < i1 ? key_of(best, at) : 0;
    const uint64_t tail = tail_at < i1 ? key_of(xt[0], tail_at) : 0;
    s_key[tid] = own > tail ? own : tail;
    if (tid == 0) s_n = 0;
    __syncthreads();
    if (tid < 64) {
        uint64_t k = s_key[tid];
#pragma unroll
        for (int w = 1; w < T / 64; w++) {
            const uint64_t u = s_key[tid + 64 * w];
            if (u > k) k = u;
        }
        k = wave_nth(k, a.top);
        if (tid == 0) s_bound = k;
    }
    Stat s = {-INFINITY, 0.0f, 0.0f};
    add(s, x);
    add(s, xt);
    s = block_join<T>(s, s_stat);
    const uint64_t bound = s_bound;  // 0: not so many lanes have any
    const auto keep = [&](uint64_t k) {
        if (k < bound || !k) return;
        const int n = atomicAdd(&s_n, 1);
        if (n < kList) s_key[n] = k;
    };
    keep(tail);
    if (own >= bound && own) {
        // by value first; the few that pass are read again, so that the code
        // for one is there once
        const float least = bound ? key_value(bound) : -INFINITY;
        hit = 0;
#pragma unroll
        for (int e = kRegs - 1; e >= 0; e--) hit = 2 * hit + !(x[e] < least);
#pragma unroll 1
        for (; hit; hit &= hit - 1) {
            const int i = index(0) + (__builtin_ctz(hit) / V) * T * V + __builtin_ctz(hit) % V;
            if ((i & ~(V - 1)) + V <= i1) keep(key_of(load1<TYPE>(a.x, x0 + i), i));
        }
    }
    __syncthreads();
    if (s_n <= kList) {
        rank_list<T>(s_key, s_n, a.top, s_top);
    } else {
        uint64_t last = ~(uint64_t)0;
#pragma unroll 1
        for (int n = 0; n < a.top; n++) {
            uint64_t k = tail < last ? tail : 0;
#pragma unroll 1
            for (int v = 0; v < kRegs / V; v++) {
                const int i = index(v * V);
                if (i + V > i1) continue;
#pragma unroll
                for (int e = 0; e < V; e++) {
                    const uint64_t u = key_of(load1<TYPE>(a.x, x0 + i + e), i + e);
                    if (u < last && u > k) k = u;
                }
            }
            last = block_max<T>(k, s_red);
            if (tid == 0) s_top[n] = last;
        }
        __syncthreads();
    }
    if (gridDim.x == 1) {
        finish<TYPE>(a, s, row, s_top);
        return;
    }
    const int64_t p = row * gridDim.x + blockIdx.x;
    if (tid == 0) a.part[p] = s;
    if (tid < a.top) a.part_key[p * a.top + tid] = s_top[tid];
}

// One block per row: the statistics of `parts` blocks, and the n largest of
// their ordered lists.  No list's n-th is above the n-th of all, so what is
// below the highest of those is dropped; the rest is ranked.  That costs two
// barriers and a second look, more than ranking up to two waves of keys: 4 lists
// of 20 for each of 64 rows 19.8 us in all, 20.5 with the bound.
template <int TYPE>
__global__ __launch_bounds__(256) void k_logprobs_join(RowArgs a, int parts) {
    constexpr int T = 256;
    __shared__ Stat s_stat[T / 64];
    __shared__ uint64_t s_red[T / 64], s_top[kTopMost], s_key[kList];
    __shared__ int s_n;
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, top = a.top;
    const uint64_t *keys = a.part_key + row * parts * top;
    Stat s = {-INFINITY, 0.0f, 0.0f};
    uint64_t bound = 0;
    // few keys are ranked as they are
    const bool few = parts * top <= kFew;
#pragma unroll 1
    for (int p = tid; p < parts; p += T) {
        join(s, a.part[row * parts + p]);
        if (top && !few) {
            const uint64_t k = keys[p * top + top - 1];
            if (k > bound) bound = k;
        }
    }
    if (few && tid < parts * top) s_key[tid] = keys[tid];
    if (tid == 0) s_n = few ? parts * top : 0;
    s = block_join<T>(s, s_stat);
    if (top) {
        if (!few) {
            bound = block_max<T>(bound, s_red);
#pragma unroll 1
            for (int i = tid; i < parts * top; i += T) {
                const uint64_t k = keys[i];
                if (k && k >= bound) {
                    const int n = atomicAdd(&s_n, 1);
                    if (n < kList) s_key[n] = k;
                }
            }
            __syncthreads();
        }
        if (s_n <= kList) {
            rank_list<T>(s_key, s_n, top, s_top);
        } else {
            uint64_t last = ~(uint64_t)0;
#pragma unroll 1
            for (int n = 0; n < top; n++) {
                uint64_t k = 0;
                for (int i = tid; i < parts * top; i += T)
                    if (keys[i] < last && keys[i] > k) k = keys[i];
                last = block_max<T>(k, s_red);
                if (tid == 0) s_top[n] = last;
            }
            __syncthreads();
        }
    }
    finish<TYPE>(a, s, row, s_top);
}

// Threads of a block and blocks of a row.  With the largest wanted, 32 elements
// a thread, and 1024 threads where a row has them: the bound, the list and the
// join cost a block the same however large it is (one row of 32,000 f32 10.6 us
// against 14.2 with 256 threads, 64 rows of 128,001 bf16 20 against 29).
// Without, a block may go on for long, and a row is shared while the grid is
// small.  1801 rows of 32,000 f32 then take 44.5 us, 5.2 TB/s; a row's time is
// that of the loads and barriers it waits for, one after another.
struct Split {
    int threads, span, parts;
};
Split split_of(int rows, int vocab, int top) {
    Split s;
    s.threads = top && vocab > 256 * kRegs ? 1024 : 256;
    const int64_t each = (int64_t)s.threads * kRegs;
    int64_t parts = (vocab + each - 1) / each;
    if (!top) parts = std::max<int64_t>(1, std::min<int64_t>(parts, 512 / rows));
    s.span = (int)((vocab + parts - 1) / parts);
    s.span = (s.span + 7) & ~7;
    s.parts = (vocab + s.span - 1) / s.span;
    return s;
}

}  // namespace

int64_t logprobs_bytes(int, int rows, int vocab, int top) {
    const Split s = split_of(rows, vocab, top);
    return s.parts == 1 ? 0 : (int64_t)rows * s.parts * (16 + 8 * (int64_t)top);
}

hipError_t launch_logprobs(int type, const void *x, int64_t ld, int rows, int vocab,
                           const int32_t *given, int n_given, float *given_lp, float *entropy,
                           int top, int32_t *top_id, float *top_lp, void *ws, hipStream_t st) {
    const Split sp = split_of(rows, vocab, top);
    uint64_t *keys = static_cast<uint64_t *>(ws);
    Stat *part = reinterpret_cast<Stat *>(keys + (sp.parts == 1 ? 0 : (int64_t)rows * sp.parts * top));
    const auto go = [&](auto type_c) {
        constexpr int TYPE = decltype(type_c)::value;
        // grid.y holds 65535 rows; more run in turns
        for (int64_t r0 = 0; r0 < rows; r0 += 65535) {
            const unsigned n = (unsigned)std::min<int64_t>(65535, rows - r0);
            const RowArgs a{static_cast<const uint8_t *>(x) + r0 * ld * (TYPE == LCMOE_TYPE_F32 ? 4 : 2),
                            ld, vocab, sp.span, given ? given + r0 * n_given : nullptr, n_given,
                            given_lp ? given_lp + r0 * n_given : nullptr, entropy ? entropy + r0 : nullptr,
                            top, top_id ? top_id + r0 * top : nullptr, top_lp ? top_lp + r0 * top : nullptr,
                            part + r0 * sp.parts, keys + r0 * sp.parts * top};
            auto *kern = !top ? k_logprobs<TYPE>
                         : sp.threads == 256 ? k_logprobs_top<TYPE, 256> : k_logprobs_top<TYPE, 1024>;
            hipLaunchKernelGGL(kern, dim3(sp.parts, n), dim3(sp.threads), 0, st, a);
            if (sp.parts > 1)
                hipLaunchKernelGGL(k_logprobs_join<TYPE>, dim3(n), dim3(256), 0, st, a, sp.parts);
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
