// Launches of the attention over a paged cache (lcmoe_kv_attention_dev): which
// tiles, and how many blocks share the context.

#include "kv_attend.h"

namespace lcmoe {

namespace {

struct Plan {
    int tiles, splits, per_seq, lo, hi, rows;  // rows of a tile
};

// blocks that share a row's context, so that about `want` blocks run and each
// has `least` steps of `st` tokens
int splits_for(const KvArgs &a, int64_t tiles, int want, int st, int least) {
    const int64_t steps = ((int64_t)a.max_pages << a.plog) / ((int64_t)st * least);
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>(128, steps));
    const int64_t base = std::max<int64_t>(1, tiles * a.KVH);
    return (int)std::max<int64_t>(1, std::min<int64_t>(most, (want + base - 1) / base));
}

// One launch (n = 1) or two: sequences of up to 16 rows, and those of more.
//
// Rows of a block: 256 (128 of heads past 128 dims) where 200 blocks of that at
// least can run, for 256 CUs, else 64, whose waves share the context.  With 32
// heads on 8 of 128 dims, 8-bit pages, 64 against 256 rows: 1400 tokens, f16
// activations (175 blocks) 54 us against 62, bf16 57 and 56; 1600 tokens (200)
// 67 against 70, bf16 72 and 65; 1600 after 10,000, bf16, 495 against 367; 3000
// tokens on 16 heads of their own (192) 87 against 113.
//
// Blocks of 16 rows share a context until 512 run: 100,000 tokens 42 us, with 256
// 41, 128 51, 2048 46; 8 sequences of 4096 20, 20, 25, 23; 64 of them 69, 71, 69,
// 88.  Blocks of 64 rows do until 256 run, where there are up to 128 at all: 64
// tokens on 30,000 68 us, with 512 77, 128 107, unshared 335; 300 on 10,000 (152
// blocks) 123 unshared, 154 shared.
int plans(const KvArgs &a, Plan (&p)[2]) {
    const int G = a.H / a.KVH;
    const int64_t most = (int64_t)a.max_new * G;  // rows of one sequence
    int n = 0;
    if (most <= 16 || (a.starts && a.n_seq > 1)) {
        p[n] = {a.n_seq, 0, 1, 0, 16, 16};
        p[n].splits = splits_for(a, a.n_seq, 512, a.i8 ? 64 : 32, kWaves);
        n++;
    }
    if (most > 16) {
        const bool alike = !a.starts || a.n_seq == 1;
        const auto tiles = [&](int M) {
            const int64_t per = (most + M - 1) / M;
            // sequences' rows fill at most this many tiles, one of each in part
            return alike ? per * a.n_seq
                         : std::min<int64_t>((int64_t)a.n_rows * G / M + a.n_seq, per * a.n_seq);
        };
        int M = a.hdp <= 128 ? 256 : 128;
        if (tiles(M) * a.KVH < 200) M = 64;
        p[n] = {(int)tiles(M), 1, alike ? (int)((most + M - 1) / M) : 0, n ? 16 : 0, INT32_MAX, M};
        if (M == 64 && p[n].tiles * a.KVH <= 128) p[n].splits = splits_for(a, p[n].tiles, 256, 64, 16);
        n++;
    }
    return n;
}

}  // namespace

int64_t kv_attention_floats(const KvArgs &a) {
    Plan p[2];
    int64_t most = 0;
    for (int i = 0, n = plans(a, p); i < n; i++)
        if (p[i].splits > 1)
            most = std::max(most, (int64_t)a.n_rows * a.H * p[i].splits * (a.hdp + 2));
    return most;
}

hipError_t launch_kv_attention(const KvArgs &a, const void *q, int64_t ldq, const float *rope,
                               float scale, void *out, int64_t ldo, float *ws,
                               hipStream_t st) {
    Plan p[2];
    for (int i = 0, n = plans(a, p); i < n; i++) {
        AttendArgs t{q, ldq, rope, scale, out, ldo, p[i].splits, p[i].per_seq, p[i].lo,
                     p[i].hi, ws, ws + (int64_t)a.n_rows * a.H * p[i].splits * a.hdp};
        if ((int64_t)p[i].tiles * a.KVH > INT32_MAX) return hipErrorInvalidConfiguration;
        const bool many = p[i].rows > 64;
        const hipError_t e = p[i].rows == 16           ? (a.i8 ? attend_i8 : attend_f16)(a, t, p[i].tiles, st)
                             : a.act == LCMOE_TYPE_F32 ? prompt_f32(a, t, p[i].tiles, many, st)
                             : a.act == LCMOE_TYPE_F16 ? prompt_f16(a, t, p[i].tiles, many, st)
                                                       : prompt_bf16(a, t, p[i].tiles, many, st);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace lcmoe
