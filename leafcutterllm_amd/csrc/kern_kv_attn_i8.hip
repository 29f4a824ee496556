// Instances of the paged attention over 8-bit pages (kv_attend.h).

#include "kv_attend.h"

namespace lcmoe {

hipError_t attend_i8(const KvArgs &a, const AttendArgs &t, int tiles, hipStream_t st) {
    return a.act == LCMOE_TYPE_F32 ? attend_launch<true, 3>(a, t, tiles, st)
                                   : attend_launch<true, 2>(a, t, tiles, st);
}

}  // namespace lcmoe
