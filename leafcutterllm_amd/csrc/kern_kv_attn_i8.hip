// Instances of the paged attention over 8-bit pages (kv_attend.h).

#include "kv_attend.h"

namespace lcmoe {

hipError_t attend_i8(const KvArgs &a, const AttendArgs &t, int tiles, bool big, hipStream_t st) {
    if (a.act == LCMOE_TYPE_F32)
        return big ? attend_launch<true, 3, kBigTile>(a, t, tiles, st)
                   : attend_launch<true, 3, 1>(a, t, tiles, st);
    return big ? attend_launch<true, 2, kBigTile>(a, t, tiles, st)
               : attend_launch<true, 2, 1>(a, t, tiles, st);
}

}  // namespace lcmoe
