// The attention kernels over paged caches for fp32 queries.
#include "kv_launch.h"

namespace lv {

int launch_tiles_f32(const Call& a, const TilePlan& p, char* ws) {
  return launch_tiles<float>(a, p, ws);
}

LV_ERROR_WORD_READER(read_errors_tiles_f32)

}  // namespace lv
