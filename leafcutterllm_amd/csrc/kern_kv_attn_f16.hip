// Instances of the paged attention over f16 pages (kv_attend.h).

#include "kv_attend.h"

namespace lcmoe {

hipError_t attend_f16(const KvArgs &a, const AttendArgs &t, int tiles, hipStream_t st) {
    // bf16 results keep 8 bits: one f16 of q and p each
    return a.act == LCMOE_TYPE_BF16 ? attend_launch<false, 1>(a, t, tiles, st)
                                    : attend_launch<false, 2>(a, t, tiles, st);
}

}  // namespace lcmoe
