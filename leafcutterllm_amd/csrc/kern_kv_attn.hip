// Launches of the attention over a paged cache (lcmoe_kv_attention_dev): which
// tiles, and how many blocks share the context.

#include "kv_attend.h"

namespace lcmoe {

namespace {

struct Plan {
    int tiles, splits, per_seq, lo, hi;
};

// blocks that share a row's context, so that about `want` blocks run
int splits_for(const KvArgs &a, int64_t tiles, int want) {
    const int64_t steps = ((int64_t)a.max_pages << a.plog) / (a.i8 ? 64 : 32) / kWaves;
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>(128, steps));
    const int64_t base = std::max<int64_t>(1, tiles * a.KVH);
    return (int)std::max<int64_t>(1, std::min<int64_t>(most, (want + base - 1) / base));
}

// One launch (n = 1) or two: sequences of up to 16 rows, and those of more.
int plans(const KvArgs &a, Plan (&p)[2]) {
    const int G = a.H / a.KVH, M = 16 * kBigTile;
    const int64_t most = (int64_t)a.max_new * G;  // rows of one sequence
    int n = 0;
    if (most <= 16 || (a.starts && a.n_seq > 1)) {
        p[n] = {a.n_seq, 0, 1, 0, 16};
        p[n].splits = splits_for(a, a.n_seq, 1024);
        n++;
    }
    if (most > 16) {
        const int per = (int)((most + M - 1) / M);
        const bool alike = !a.starts || a.n_seq == 1;
        // sequences' rows fill at most this many tiles, one of each in part
        const int64_t tiles = alike ? (int64_t)per * a.n_seq
                                    : std::min<int64_t>((int64_t)a.n_rows * G / M + a.n_seq,
                                                        (int64_t)per * a.n_seq);
        p[n] = {(int)tiles, 0, alike ? per : 0, n ? 16 : 0, INT32_MAX};
        p[n].splits = splits_for(a, tiles, 512);
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
                               float scale, void *out, int64_t ldo, bool vec, float *ws,
                               hipStream_t st) {
    Plan p[2];
    for (int i = 0, n = plans(a, p); i < n; i++) {
        AttendArgs t{q, ldq, rope, scale, out, ldo, vec, p[i].splits, p[i].per_seq, p[i].lo,
                     p[i].hi, ws, ws + (int64_t)a.n_rows * a.H * p[i].splits * a.hdp};
        const bool big = p[i].hi > 16;
        const hipError_t e = a.i8 ? attend_i8(a, t, p[i].tiles, big, st)
                                  : attend_f16(a, t, p[i].tiles, big, st);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace lcmoe
