// What keeps the attention over the 4-bit cache inside its memory when a wait gives up, for the tests.
#include "kv4_attention_tc.cuh"

#define EXPORT extern "C" __attribute__((visibility("default")))

EXPORT int valid_record(int first_part, int last_warp, int list_warps)
{
    return lun::kv4_valid_record(first_part, last_warp, list_warps);
}
