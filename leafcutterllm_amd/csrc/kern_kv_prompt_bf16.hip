// Instances of the prompts' attention for bf16 activations (kv_prompt.h).

#include "kv_prompt.h"

namespace lcmoe {

hipError_t prompt_bf16(const KvArgs &a, const AttendArgs &t, int tiles, bool many, hipStream_t st) {
    return prompt_launch<LCMOE_TYPE_BF16>(a, t, tiles, many, st);
}

}  // namespace lcmoe
