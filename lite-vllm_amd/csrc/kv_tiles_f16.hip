// The attention kernels over paged caches for f16 queries.
#include "kv_launch.h"

namespace lv {

int launch_tiles_f16(const Call& a, const TilePlan& p, char* ws) {
  return launch_tiles<f16>(a, p, ws);
}

LV_ERROR_WORD_READER(read_errors_tiles_f16)

}  // namespace lv
