// Instances of the paged attention over f16 pages (kv_attend.h).

#include "kv_attend.h"

namespace lcmoe {

hipError_t attend_f16(const KvArgs &a, const AttendArgs &t, int tiles, bool big, hipStream_t st) {
    // bf16 results keep 8 bits: one f16 of q and p each
    if (a.act == LCMOE_TYPE_BF16)
        return big ? attend_launch<false, 1, kBigTile>(a, t, tiles, st)
                   : attend_launch<false, 1, 1>(a, t, tiles, st);
    return big ? attend_launch<false, 2, kBigTile>(a, t, tiles, st)
               : attend_launch<false, 2, 1>(a, t, tiles, st);
}

}  // namespace lcmoe
