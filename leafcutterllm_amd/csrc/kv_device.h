// The paged K/V cache's layout and batch, shared by its kernels.
//
// A page holds, per K/V head, page_tokens / 16 units of 16 tokens, each 16 *
// hdp values (hdp: head_dim rounded up to 32, past 128 to
// 64) in the order in which a wave of
// the attention feeds its matrix instructions, so that a unit is read with
// 16-byte loads, 1 KiB in a row:
//   K, "narrow" (f16, and the last 32 dims in 8 bits when hdp % 64 == 32):
//     for each 32 dims [4 groups of 8 dims][16 tokens][8 dims];
//   K, "wide" (8 bits): for each 64 dims [4 groups of 16 dims][16 tokens][16];
//   V, narrow: for each 32 dims [4 groups of 4 tokens][16 dims][2][4 tokens],
//     the [2] being dims 16 apart;
//   V, wide: for each 64 dims [4 groups of 4 tokens][16 dims][4][4 tokens].
#pragma once

#include <cmath>

#include "device_common.h"
#include "kernels.h"

namespace lcmoe {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx2 __attribute__((ext_vector_type(2)));

// place of (token r of the unit, dim d); 8 dims from a multiple of 8 are
// contiguous
template <bool I8>
__device__ __forceinline__ int k_place(int hdp, int r, int d) {
    if (I8 && d < (hdp & ~63)) return (d >> 6) * 1024 + ((d >> 4) & 3) * 256 + r * 16 + (d & 15);
    return (d >> 5) * 512 + ((d >> 3) & 3) * 128 + r * 8 + (d & 7);
}
// 4 tokens from a multiple of 4 are contiguous
template <bool I8>
__device__ __forceinline__ int v_place(int hdp, int r, int d) {
    const int t = d >> 4;
    if (I8 && d < (hdp & ~63))
        return (t >> 2) * 1024 + (r >> 2) * 256 + (d & 15) * 16 + (t & 3) * 4 + (r & 3);
    return (t >> 1) * 512 + (r >> 2) * 128 + (d & 15) * 8 + (t & 1) * 4 + (r & 3);
}
// first value of a unit, counted in values of the pool
__device__ __forceinline__ int64_t unit_base(const KvArgs &a, int page, int h, int unit) {
    return ((((int64_t)page * a.KVH + h) << (a.plog - 4)) + unit) * 16 * a.hdp;
}

// byte `B` of four words, as one word
template <int B>
__device__ __forceinline__ uint32_t bytes4(const uint32_t (&x)[4]) {
    constexpr uint32_t pair = 0x0c0c0000u | (uint32_t)(B + 4) << 8 | B;
    const uint32_t a = __builtin_amdgcn_perm(x[1], x[0], pair);
    const uint32_t b = __builtin_amdgcn_perm(x[3], x[2], pair);
    return __builtin_amdgcn_perm(b, a, 0x05040100u);
}

// Sequence b of the batch: its first row, cached tokens and new tokens, held
// inside the call's rows and the page table whatever the device arrays say
// (tokens past the table's capacity are dropped).
struct Seq {
    int row0, len0, cnt;
};
__device__ __forceinline__ Seq sequence(const KvArgs &a, int b) {
    int r0, r1;
    if (a.starts) {
        r0 = min(max(a.starts[b], 0), a.n_rows);
        r1 = min(max(a.starts[b + 1], r0), a.n_rows);
    } else {
        r0 = b * a.max_new;
        r1 = r0 + a.max_new;
    }
    const int cap = a.max_pages << a.plog;
    const int len0 = min(max(a.lens[b], 0), cap);
    return {r0, len0, min(min(r1 - r0, a.max_new), cap - len0)};
}

// Work item `tile` of a batch whose sequence b has count(sequence b) of them:
// its sequence (-1 past the last) and number inside it.  Every wave of a block
// finds it for itself, 64 sequences at a time; wave-uniform results.
template <class Count>
__device__ __forceinline__ int find_tile(const KvArgs &a, int tile, Count count, int &j) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int b0 = 0; b0 < a.n_seq; b0 += 64) {
        const int b = b0 + lane;
        int s = b < a.n_seq ? count(sequence(a, b)) : 0;
        const int own = s;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int u = __shfl_up(s, o, 64);
            if (lane >= o) s += u;
        }
        const uint64_t hit = __ballot(tile < before + s);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            j = __builtin_amdgcn_readfirstlane(tile - before - __shfl(s - own, l, 64));
            return b0 + l;
        }
        before += __shfl(s, 63, 64);
    }
    return -1;
}

// N (4 or 8) consecutive activations (f32, f16 or bf16) from element e of
// `base`, which need be aligned to an element only
template <int ACT, int N>
__device__ __forceinline__ void load_n(const void *base, int64_t e, float (&o)[N]) {
    if constexpr (ACT == LCMOE_TYPE_F32) {
        __builtin_memcpy(o, static_cast<const float *>(base) + e, 4 * N);
    } else {
        uint32_t w[N / 2];
        __builtin_memcpy(w, static_cast<const uint16_t *>(base) + e, 2 * N);
#pragma unroll
        for (int i = 0; i < N / 2; i++) {
            if constexpr (ACT == LCMOE_TYPE_F16) {
                o[2 * i] = dh2f(w[i] & 0xffff);
                o[2 * i + 1] = dh2f(w[i] >> 16);
            } else {
                o[2 * i] = __uint_as_float(w[i] << 16);
                o[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        }
    }
}

// f32 to bf16, to nearest even (NaN stays NaN)
__device__ __forceinline__ uint32_t to_bf16(float f) {
    return __builtin_bit_cast(uint16_t, (__bf16)f);
}
template <int ACT>
__device__ __forceinline__ uint32_t to16(float f) {
    if constexpr (ACT == LCMOE_TYPE_F16) {
        const _Float16 h = (_Float16)f;
        uint16_t b;
        __builtin_memcpy(&b, &h, 2);
        return b;
    } else {
        return to_bf16(f);
    }
}
template <int ACT, int N>
__device__ __forceinline__ void store_n(void *base, int64_t e, const float (&o)[N]) {
    if constexpr (ACT == LCMOE_TYPE_F32) {
        __builtin_memcpy(static_cast<float *>(base) + e, o, 4 * N);
    } else {
        uint32_t w[N / 2];
#pragma unroll
        for (int i = 0; i < N / 2; i++) w[i] = to16<ACT>(o[2 * i]) | (to16<ACT>(o[2 * i + 1]) << 16);
        __builtin_memcpy(static_cast<uint16_t *>(base) + e, w, 2 * N);
    }
}

}  // namespace lcmoe
