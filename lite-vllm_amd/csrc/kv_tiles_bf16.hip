// The attention kernels over paged caches for bf16 queries.
#include "kv_launch.h"

namespace lv {

int launch_tiles_bf16(const Call& a, const TilePlan& p, char* ws) {
  return launch_tiles<bf16>(a, p, ws);
}

LV_ERROR_WORD_READER(read_errors_tiles_bf16)

}  // namespace lv
